// Rotary positions of many tokens: whole heads or their first dims, half or interleaved pairs,
// any frequencies.
//
// An angle is position x frequency, formed in binary64 in turns and reduced there (t - rint(t)),
// since a binary32 product of a position near 10^6 is off by 0.06 radians; sine and cosine of the
// reduced angle are then taken in binary32.  A workgroup forms the rotary/2 angles of its tokens
// once, in LDS, for all heads.
#include "tt_abi_internal.h"
#include "tt_common.h"

namespace tt {

// Eight elements of a 16-byte aligned piece (two pieces of binary32).
template <typename T> __device__ __forceinline__ void load8(const T* p, float x[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = piece_f32<T>(v, e);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float x[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float x[8]) {
  *reinterpret_cast<uint4*>(p) = pack_piece<T>(x);
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float x[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

struct RotaryParams {
  const void* x[2];        // q, k
  void* out[2];
  int64_t x_token[2], x_head[2], o_token[2], o_head[2];
  int heads[2];
  const void* positions;
  int position_shift;      // log2 of the position's size in 32-bit words
  const double* inv_freq;
  float amplitude;
  int64_t tokens;
  int head_dim, rotary;
};

// One thread per pair or copied dim: any sizes, strides and alignment.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams P) {
  extern __shared__ float2 turn[];
  const int64_t token = blockIdx.x;
  const int half = P.rotary >> 1, copies = P.head_dim - P.rotary;
  const int64_t pos = load_expert(P.positions, P.position_shift, token);
  for (int i = threadIdx.x; i < half; i += 256) {
    const double t = (double)pos * P.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &s, &c);
    turn[i] = make_float2(c * P.amplitude, s * P.amplitude);
  }
  __syncthreads();
  const int units = half + copies;
  for (int w = 0; w < 2; w++) {
    for (int u = threadIdx.x; u < P.heads[w] * units; u += 256) {
      const int h = u / units, i = u - h * units;
      const T* x = reinterpret_cast<const T*>(P.x[w]) + token * P.x_token[w] + h * P.x_head[w];
      T* o = reinterpret_cast<T*>(P.out[w]) + token * P.o_token[w] + h * P.o_head[w];
      if (i < half) {
        const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : i + half;
        const float a = to_f32(x[ia]), b = to_f32(x[ib]);
        const float2 cs = turn[i];
        store<T>(o + ia, a * cs.x - b * cs.y);
        store<T>(o + ib, b * cs.x + a * cs.y);
      } else {
        o[half + i] = x[half + i];
      }
    }
  }
}

// Rows whose parts start on 16-byte boundaries and come in whole pieces of eight dims: a thread takes
// eight pairs of the half layout (two pieces) or four of the interleaved one, or copies a piece.
// `tokens_per` tokens share a workgroup where one has few pieces.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_vec_kernel(RotaryParams P, int tokens_per) {
  extern __shared__ __attribute__((aligned(16))) float turn_s[];   // cosines, then sines, of each token
  const int half = P.rotary >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * tokens_per;
  const int tokens = (int)min((int64_t)tokens_per, P.tokens - t0);
  for (int u = threadIdx.x; u < tokens * half; u += 256) {
    const int tk = u / half, i = u - tk * half;
    const double t = (double)load_expert(P.positions, P.position_shift, t0 + tk) * P.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &s, &c);
    turn_s[tk * P.rotary + i] = c * P.amplitude;
    turn_s[tk * P.rotary + half + i] = s * P.amplitude;
  }
  __syncthreads();
  const int turns = INTERLEAVED ? P.rotary / 8 : half / 8;
  const int units = turns + (P.head_dim - P.rotary) / 8;
  const int heads = P.heads[0] + P.heads[1];
  for (int w = threadIdx.x; w < tokens * heads * units; w += 256) {
    const int hu = w / units, u = w - hu * units;
    const int tk = hu / heads, hh = hu - tk * heads;
    const bool second = hh >= P.heads[0];
    const int h = second ? hh - P.heads[0] : hh;
    const T* x = reinterpret_cast<const T*>(second ? P.x[1] : P.x[0]) + (t0 + tk) * (second ? P.x_token[1] : P.x_token[0]) +
                 h * (second ? P.x_head[1] : P.x_head[0]);
    T* o = reinterpret_cast<T*>(second ? P.out[1] : P.out[0]) + (t0 + tk) * (second ? P.o_token[1] : P.o_token[0]) +
           h * (second ? P.o_head[1] : P.o_head[0]);
    const float* cs = turn_s + tk * P.rotary;
    if (u >= turns) {
      const int d = P.rotary + 8 * (u - turns);
      if (x != o) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; k++) reinterpret_cast<uint4*>(o + d)[k] = reinterpret_cast<const uint4*>(x + d)[k];
      }
    } else if (INTERLEAVED) {
      float a[8], r[8];
      load8<T>(x + 8 * u, a);
      const float4 c = *reinterpret_cast<const float4*>(cs + 4 * u), s = *reinterpret_cast<const float4*>(cs + half + 4 * u);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        r[2 * k] = a[2 * k] * cc[k] - a[2 * k + 1] * ss[k];
        r[2 * k + 1] = a[2 * k + 1] * cc[k] + a[2 * k] * ss[k];
      }
      store8<T>(o + 8 * u, r);
    } else {
      float a[8], b[8], ra[8], rb[8];
      load8<T>(x + 8 * u, a);
      load8<T>(x + half + 8 * u, b);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float c = cs[8 * u + k], s = cs[half + 8 * u + k];
        ra[k] = a[k] * c - b[k] * s;
        rb[k] = b[k] * c + a[k] * s;
      }
      store8<T>(o + 8 * u, ra);
      store8<T>(o + half + 8 * u, rb);
    }
  }
}

template <typename T>
static int launch_rotary(const RotaryParams& P, bool interleaved, hipStream_t st) {
  constexpr uintptr_t step = 16 / sizeof(T);
  bool vec = P.head_dim % 8 == 0 && P.rotary % (interleaved ? 8 : 16) == 0;
  for (int w = 0; w < (P.heads[1] > 0 ? 2 : 1); w++)
    vec = vec && aligned(P.x[w], 16) && aligned(P.out[w], 16) &&
          ((P.x_token[w] | P.x_head[w] | P.o_token[w] | P.o_head[w]) & (int64_t)(step - 1)) == 0;
  if (vec) {
    // a round of the workgroup's threads, at most eight tokens
    const int pieces = (P.heads[0] + P.heads[1]) * ((interleaved ? P.rotary / 8 : P.rotary / 16) + (P.head_dim - P.rotary) / 8);
    int per = 256 / pieces;
    per = per < 1 ? 1 : per > 8 ? 8 : per;
    const dim3 grid((unsigned)((P.tokens + per - 1) / per));
    const size_t lds = sizeof(float) * (size_t)(per * P.rotary);
    if (interleaved) hipLaunchKernelGGL((rotary_vec_kernel<T, true>), grid, dim3(256), lds, st, P, per);
    else hipLaunchKernelGGL((rotary_vec_kernel<T, false>), grid, dim3(256), lds, st, P, per);
    return check_launch("rotary_rows");
  }
  const dim3 grid((unsigned)P.tokens), block(256);
  const size_t lds = sizeof(float2) * (size_t)(P.rotary / 2);
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, true>), grid, block, lds, st, P);
  else hipLaunchKernelGGL((rotary_kernel<T, false>), grid, block, lds, st, P);
  return check_launch("rotary_rows");
}

}  // namespace tt

using namespace tt;

extern "C" int tt_rotary_rows(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                              int64_t k_head, int dtype, const void* positions, int position_bytes,
                              const double* inv_freq, float amplitude, int interleaved, int64_t tokens, int64_t heads,
                              int64_t kv_heads, int64_t head_dim, int64_t rotary, void* q_out, int64_t qo_token,
                              int64_t qo_head, void* k_out, int64_t ko_token, int64_t ko_head, void* stream) {
  const char* what = "rotary_rows";
  TT_REQUIRE(tokens >= 0 && tokens < (1LL << 31), "%s: bad token count", what);
  TT_REQUIRE(heads > 0 && kv_heads >= 0 && heads <= 65536 && kv_heads <= 65536, "%s: bad head counts", what);
  TT_REQUIRE(head_dim > 0 && head_dim <= 1024 && rotary > 0 && rotary <= head_dim && rotary % 2 == 0,
             "%s: rotary dims must be even and at most head_dim (1024 at most)", what);
  TT_REQUIRE(valid_out_dtype(dtype), "%s: dtype must be fp16, bf16 or fp32", what);
  if (tokens == 0) return TT_OK;
  RotaryParams P{};
  TT_REQUIRE(index_shift(position_bytes, &P.position_shift), "%s: positions must be int32 or int64", what);
  TT_REQUIRE(q && q_out && positions && inv_freq && (kv_heads == 0 || (k && k_out)), "%s: null pointer", what);
  P.x[0] = q; P.x[1] = k; P.out[0] = q_out; P.out[1] = k_out;
  P.x_token[0] = q_token; P.x_token[1] = k_token; P.x_head[0] = q_head; P.x_head[1] = k_head;
  P.o_token[0] = qo_token; P.o_token[1] = ko_token; P.o_head[0] = qo_head; P.o_head[1] = ko_head;
  P.heads[0] = (int)heads; P.heads[1] = (int)kv_heads;
  P.positions = positions; P.inv_freq = inv_freq; P.amplitude = amplitude;
  P.tokens = tokens; P.head_dim = (int)head_dim; P.rotary = (int)rotary;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TT_F16) return launch_rotary<f16_t>(P, interleaved != 0, st);
  if (dtype == TT_BF16) return launch_rotary<bf16_t>(P, interleaved != 0, st);
  return launch_rotary<float>(P, interleaved != 0, st);
}
