// Eight consecutive elements of a row that starts on a 16-byte boundary.
#pragma once

#include "tt_common.h"

namespace tt {

// Eight elements as they are stored: one 16-byte piece, two of binary32.
template <typename T> struct Eight {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ float get(int e) const { return piece_f32<T>(v, e); }
  __device__ __forceinline__ void set(const float* x) { v = pack_piece<T>(x); }
};
template <> struct Eight<float> {
  float x[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ float get(int e) const { return x[e]; }
  __device__ __forceinline__ void set(const float* y) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = y[e];
  }
};

}  // namespace tt
