// Rotary positions of many tokens: whole heads or their first dims, half or interleaved pairs,
// any frequencies.
//
// An angle is position x frequency, formed in binary64 in turns and reduced there (t - rint(t)),
// since a binary32 product of a position near 10^6 is off by 0.06 radians; sine and cosine of the
// reduced angle are then taken in binary32.  A workgroup forms the rotary/2 angles of its tokens
// once, in LDS, for all heads, while the vectors are on their way: what bounds it is memory (8191 tokens
// of 72 heads of 128, 302 MB: 62 us, 4.9 TB/s; a thread per pair 141).
#include "tt_abi_internal.h"
#include "tt_common.h"
#include "tt_eight.h"
#include "tt_regions.h"

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

// Rows whose parts start on 16-byte boundaries and come in whole pieces of eight dims: a thread keeps
// one place of the head -- eight pairs of the half layout (two pieces), four of the interleaved one, or
// a piece to copy -- and walks over the heads of its workgroup's tokens (`tokens_per`, more than one
// where a token has few pieces), kAhead at a time: requested together, the first before the angles are
// formed, and written together, because a load that was issued after a store waits for it.
constexpr int kAhead = 4;
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(1024) void rotary_vec_kernel(RotaryParams P, int tokens_per, int units) {
  extern __shared__ __attribute__((aligned(16))) float turn_s[];   // cosines, then sines, of each token
  constexpr int NP = INTERLEAVED ? 1 : 2;      // pieces of a place
  const int half = P.rotary >> 1;
  const int turns = INTERLEAVED ? P.rotary / 8 : half / 8;
  const int64_t t0 = (int64_t)blockIdx.x * tokens_per;
  const int tokens = (int)min((int64_t)tokens_per, P.tokens - t0);
  const int heads = P.heads[0] + P.heads[1];
  const int rows = (int)blockDim.x / units;                // heads in flight
  const int r0 = (int)threadIdx.x / units, u = (int)threadIdx.x - r0 * units;
  const int total = r0 < rows ? tokens * heads : 0;
  const bool copy = u >= turns;
  const int d0 = copy ? P.rotary + 8 * (u - turns) : 8 * u, d1 = INTERLEAVED || copy ? d0 : d0 + half;
  struct Place {
    const T* x;
    T* o;
    int token;
  };
  auto place = [&](int r) __attribute__((always_inline)) {
    const int tk = tokens_per == 1 ? 0 : r / heads, hh = r - tk * heads;
    const bool second = hh >= P.heads[0];
    const int h = second ? hh - P.heads[0] : hh;
    return Place{reinterpret_cast<const T*>(second ? P.x[1] : P.x[0]) + (t0 + tk) * (second ? P.x_token[1] : P.x_token[0]) +
                     h * (second ? P.x_head[1] : P.x_head[0]),
                 reinterpret_cast<T*>(second ? P.out[1] : P.out[0]) + (t0 + tk) * (second ? P.o_token[1] : P.o_token[0]) +
                     h * (second ? P.o_head[1] : P.o_head[0]), tk};
  };
  Eight<T> a[kAhead], b[kAhead];
  auto load = [&](int r) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (r + k * rows < total) {
        const Place p = place(r + k * rows);
        a[k].load(p.x + d0);
        if (NP == 2 && !copy) b[k].load(p.x + d1);
      }
  };
  load(r0);
  for (int v = threadIdx.x; v < tokens * half; v += (int)blockDim.x) {
    const int tk = tokens_per == 1 ? 0 : v / half, i = v - tk * half;
    const double t = (double)load_expert(P.positions, P.position_shift, t0 + tk) * P.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &s, &c);
    turn_s[tk * P.rotary + i] = c * P.amplitude;
    turn_s[tk * P.rotary + half + i] = s * P.amplitude;
  }
  lds_barrier();
  for (int r = r0; r < total; r += kAhead * rows) {
    if (r != r0) load(r);
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      if (r + k * rows >= total) break;
      const Place p = place(r + k * rows);
      if (!copy) {
        const float* cs = turn_s + p.token * P.rotary;
        float ra[8], rb[8];
        if (INTERLEAVED) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float c = cs[4 * u + e], s = cs[half + 4 * u + e];
            const float x = a[k].get(2 * e), y = a[k].get(2 * e + 1);
            ra[2 * e] = x * c - y * s;
            ra[2 * e + 1] = y * c + x * s;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float c = cs[8 * u + e], s = cs[half + 8 * u + e];
            const float x = a[k].get(e), y = b[k].get(e);
            ra[e] = x * c - y * s;
            rb[e] = y * c + x * s;
          }
          b[k].set(rb);
          b[k].store(p.o + d1);
        }
        a[k].set(ra);
      }
      // one store for turned and copied pieces of a wave (in place, a copied one is what it was)
      a[k].store(p.o + d0);
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
    const int units = (interleaved ? P.rotary / 8 : P.rotary / 16) + (P.head_dim - P.rotary) / 8;   // 128 at most
    const int64_t pieces = (int64_t)units * (P.heads[0] + P.heads[1]);
    // Few pieces: a thread for each.  Many: kAhead for each thread, so that every load comes before the
    // first store (8191 tokens of 72 heads of 128, 64 dims turned: 256 threads, which take some pieces in a
    // second turn, 67.8 us, 320 without one 65.6; 61.8, 4.9 TB/s, since turned and copied pieces share a
    // store).  Several tokens together where a token has few (4096 tokens of 3 heads of 64: 5.0 us with
    // one token per workgroup, 4.0 with eight).
    const bool many = P.tokens * pieces > (int64_t)kAhead * 256 * device_cus();
    int64_t per = (many ? 1024 : P.tokens >= 1024 ? 256 : 0) / pieces;
    per = per < 1 ? 1 : per > 8 ? 8 : per;
    int64_t threads = (per * pieces + (many ? kAhead : 1) - 1) / (many ? kAhead : 1);
    threads = (threads + units - 1) / units * units;
    threads = threads < 64 ? 64 : threads > 960 ? 960 : (threads + 63) / 64 * 64;
    const dim3 grid((unsigned)((P.tokens + per - 1) / per)), block((unsigned)threads);
    const size_t lds = sizeof(float) * (size_t)(per * P.rotary);
    if (interleaved) hipLaunchKernelGGL((rotary_vec_kernel<T, true>), grid, block, lds, st, P, (int)per, units);
    else hipLaunchKernelGGL((rotary_vec_kernel<T, false>), grid, block, lds, st, P, (int)per, units);
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
  TT_REQUIRE(tokens >= 0 && tokens <= (1 << 22), "%s: at most 2^22 tokens", what);
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
  // an output has one writer for each place, and nobody else's input there
  const int64_t element = dtype == TT_F32 ? 4 : 2;
  const Region in[2] = {{q, element, head_dim, {{tokens, q_token}, {heads, q_head}}},
                        {k, element, head_dim, {{tokens, k_token}, {kv_heads, k_head}}}};
  const Region made[2] = {{q_out, element, head_dim, {{tokens, qo_token}, {heads, qo_head}}},
                          {k_out, element, head_dim, {{tokens, ko_token}, {kv_heads, ko_head}}}};
  TT_REQUIRE(made[0].once() && made[1].once() && apart(made[0], made[1]), "%s: tokens and heads that are written must not share memory", what);
  for (int w = 0; w < 2; w++)
    TT_REQUIRE((made[w].same(in[w]) || apart(made[w], in[w])) && apart(made[w], in[1 - w]),
               "%s: an output may be its input, but share no memory with one otherwise", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TT_F16) return launch_rotary<f16_t>(P, interleaved != 0, st);
  if (dtype == TT_BF16) return launch_rotary<bf16_t>(P, interleaved != 0, st);
  return launch_rotary<float>(P, interleaved != 0, st);
}
