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

template <typename T>
static int launch_rotary(const RotaryParams& P, bool interleaved, hipStream_t st) {
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
