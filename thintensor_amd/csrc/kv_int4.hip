// Packing tokens into the 4-bit KV cache and reading them back (layout and rounding: tt_int4_cache
// and tt_kv_append_int4 in thintensor_hip.h).
//
// A workgroup owns one block of eight cache tokens of one sequence and KV head: the V words hold
// eight tokens, so a word has one writer, which merges the tokens it was not given from memory.  Half
// of its threads pack K, half V; a thread holds eight dims of one token, and a group's extremes are
// exact under any order, taken over its 4, 8 or 16 lanes.
#include "kv_int4.h"
#include "tt_common.h"
#include "tt_eight.h"

namespace tt {

struct KvRowsParams {
  tt_int4_cache c;
  void* x[2];              // k, v
  int64_t x_row[2], x_token[2], x_head[2];
  const int32_t* starts;
  const int32_t* counts;
  int tokens, vec;         // vec: eight elements of k and v start on 16-byte boundaries
};

// The exact decisions below are made in binary64, where hi - m, x - m and what a code leaves of them are
// exact.  They are only reached next to a border: binary32 is off by less than 2^-18 of a step, and
// whatever is further than that from a border has the same answer there.

// The smallest s of seven significant bits with 15 s >= hi - m; a division only proposes it.
__device__ __noinline__ float exact_step(float hi, float m) {
  const double reach = (double)hi - (double)m;
  if (!(reach > 0.0)) return 0.0f;
  const double raw = reach / 15.0;
  int e = (int)((__builtin_bit_cast(uint64_t, raw) >> 52) & 2047) - 1022 - 7;   // lsb of 7 bits
  if (e < -24) e = -24;
  const double lsb = __builtin_bit_cast(double, (uint64_t)(e + 1023) << 52);
  double s = __builtin_ceil(raw / lsb) * lsb;
  if (15.0 * (s - lsb) >= reach) s -= lsb;
  if (15.0 * s < reach) s += lsb;
  return (float)__builtin_fmin(s, 4064.0);
}

// (x - m) / s to the nearest code, ties to even: the product with 1/s proposes, the residual decides.
__device__ __noinline__ uint32_t exact_code(float x, float m, float s) {
  const double d = (double)x - (double)m, sd = (double)s;
  double q = __builtin_rint(d / sd);
  const double r2 = 2.0 * __builtin_fma(-q, sd, d);
  const bool odd = ((int64_t)q & 1) != 0;
  if (r2 > sd || (r2 == sd && odd)) q += 1.0;
  else if (r2 < -sd || (r2 == -sd && odd)) q -= 1.0;
  return (uint32_t)(int)__builtin_fmin(__builtin_fmax(q, 0.0), 15.0);
}

// A group's m and s from its extremes.
__device__ __forceinline__ float group_step(float hi, float m) {
  const float raw = (hi - m) * (1.0f / 15.0f);
  int e = (int)((__builtin_bit_cast(uint32_t, raw) >> 23) & 255) - 126 - 7;   // lsb of 7 bits
  if (e < -24) e = -24;
  const float t = __builtin_amdgcn_ldexpf(raw, -e);                           // at most 128
  const float n = __builtin_ceilf(t);
  // next to a whole number of units, or where the range is none or past the format's end
  if (!(n - t > 0x1p-10f && n - t < 1.0f - 0x1p-10f && raw < 4000.0f)) return exact_step(hi, m);
  return __builtin_amdgcn_ldexpf(n, e);
}

__device__ __forceinline__ uint32_t code_of(float x, float m, float s, float inv) {
  const float y = (x - m) * inv;
  const float q = __builtin_rintf(y);
  if (__builtin_expect(__builtin_fabsf(y - q) > 0.5f - 0x1p-12f, 0)) return exact_code(x, m, s);
  return (uint32_t)(int)__builtin_fminf(__builtin_fmaxf(q, 0.0f), 15.0f);
}

template <int G>   // over G / 8 neighbouring lanes
__device__ __forceinline__ void group_extremes(float& lo, float& hi, float& poison) {
#define TT_LEVEL(M)                                   \
  if (G / 8 > M) {                                    \
    lo = __builtin_fminf(lo, xor_partner<M>(lo));     \
    hi = __builtin_fmaxf(hi, xor_partner<M>(hi));     \
    poison = poison + xor_partner<M>(poison);         \
  }
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8)
#undef TT_LEVEL
}

template <typename T, int D, int G>
__global__ __launch_bounds__(2 * D) void kv_append_int4_kernel(KvRowsParams P) {
  constexpr int W = D / 8;                         // words (and lanes) per token
  constexpr int NG = D / G;
  __shared__ uint32_t vw[8][W];
  const int row = blockIdx.z, head = blockIdx.y;
  const int start = P.starts[row];
  const int count = P.counts ? min(P.counts[row], P.tokens) : P.tokens;
  const int64_t block = (int64_t)(start >> 3) + blockIdx.x;
  const int which = threadIdx.x / D;               // 0: K, 1: V
  const int tid = threadIdx.x % D;
  const int token = tid / W, word = tid % W;
  const int64_t pos = 8 * block + token;
  const int64_t t = pos - start;
  const bool valid = t >= 0 && t < count && pos >= 0 && pos < P.c.capacity;
  float x[8];
  const T* src = reinterpret_cast<const T*>(P.x[which]) + row * P.x_row[which] + (valid ? t : 0) * P.x_token[which] +
                 head * P.x_head[which] + 8 * word;
  if (P.vec) {
    Eight<T> v;
    v.load(src);
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = valid ? v.get(e) : 0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = valid ? to_f32(src[e]) : 0.0f;
  }
  float lo = x[0], hi = x[0], poison = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    lo = __builtin_fminf(lo, x[e]);
    hi = __builtin_fmaxf(hi, x[e]);
    poison += x[e] * 0.0f;                         // NaN where x is not finite
  }
  group_extremes<G>(lo, hi, poison);
  const bool finite = poison == poison;
  const float m = round_f16(__builtin_fminf(__builtin_fmaxf(lo, -65504.0f), 65504.0f));
  const float s = finite ? group_step(hi, m) : 0.0f;
  // a group that is not finite reads as NaN
  const uint16_t mb = finite ? f32_to_f16_bits(m) : 0x7e00u, sb = finite ? f32_to_f16_bits(s) : 0x7e00u;
  uint32_t codes = 0;
  if (s > 0.0f) {
    const float inv = 1.0f / s;
#pragma unroll
    for (int e = 0; e < 8; e++) codes |= code_of(x[e], m, s, inv) << (4 * e);
  }
  if (which == 0) {
    if (valid) {
      const int64_t at = row * P.c.kc_seq + head * P.c.kc_head + pos * W + word;
      reinterpret_cast<uint32_t*>(P.c.k_codes)[at] = codes;
      if (word % (G / 8) == 0) {
        const int64_t sat = row * P.c.ks_seq + head * P.c.ks_head + (pos * NG + word / (G / 8)) * 2;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(P.c.k_scales) + sat) = sb | ((uint32_t)mb << 16);
      }
    }
  } else {
    vw[token][word] = codes;
    if (valid && word % (G / 8) == 0) {
      uint16_t* vs = reinterpret_cast<uint16_t*>(P.c.v_scales) + row * P.c.vs_seq + head * P.c.vs_head +
                     ((block * NG + word / (G / 8)) * 2) * 8 + token;
      vs[0] = sb;
      vs[8] = mb;
    }
  }
  __syncthreads();
  if (which == 0 || block < 0 || block >= P.c.capacity / 8) return;
  // this thread's dim of the eight tokens; the tokens that were not given keep their codes
  const int d = tid;
  uint32_t word_out = 0, keep = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int64_t pk = 8 * block + k, tk = pk - start;
    const int nib = 4 * ((k >> 1) + 4 * (k & 1));
    if (tk >= 0 && tk < count) word_out |= ((vw[k][d / 8] >> (4 * (d % 8))) & 15u) << nib;
    else keep |= 15u << nib;
  }
  if (keep == 0xffffffffu) return;
  uint32_t* dst = reinterpret_cast<uint32_t*>(P.c.v_codes) + row * P.c.vc_seq + head * P.c.vc_head + block * D + d;
  if (keep) word_out |= *dst & keep;
  *dst = word_out;
}

template <typename T, int D, int G>
__global__ __launch_bounds__(2 * D) void kv_read_int4_kernel(KvRowsParams P) {
  constexpr int W = D / 8;
  constexpr int NG = D / G;
  const int row = blockIdx.z, head = blockIdx.y;
  const int start = P.starts[row];
  const int count = P.counts ? min(P.counts[row], P.tokens) : P.tokens;
  const int64_t block = (int64_t)(start >> 3) + blockIdx.x;
  const int which = threadIdx.x / D;
  const int tid = threadIdx.x % D;
  const int token = tid / W, word = tid % W;
  const int64_t pos = 8 * block + token;
  const int64_t t = pos - start;
  if (!(t >= 0 && t < count && pos >= 0 && pos < P.c.capacity)) return;
  T* dst = reinterpret_cast<T*>(P.x[which]) + row * P.x_row[which] + t * P.x_token[which] + head * P.x_head[which] + 8 * word;
  float y[8];
  if (which == 0) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(P.c.k_codes)[row * P.c.kc_seq + head * P.c.kc_head + pos * W + word];
    const uint32_t sm = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(P.c.k_scales) + row * P.c.ks_seq +
                                                           head * P.c.ks_head + (pos * NG + word / (G / 8)) * 2);
    const float s = lo_f32<f16_t>(sm), m = hi_f32<f16_t>(sm);
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)((w >> (4 * e)) & 15u), s, m);
  } else {
    const uint4* vc = reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(P.c.v_codes) + row * P.c.vc_seq +
                                                     head * P.c.vc_head + block * D + 8 * word);
    const uint4 w0 = vc[0], w1 = vc[1];
    const f16_t* vs = reinterpret_cast<const f16_t*>(P.c.v_scales) + row * P.c.vs_seq + head * P.c.vs_head +
                      ((block * NG + word / (G / 8)) * 2) * 8 + token;
    const float s = to_f32(vs[0]), m = to_f32(vs[8]);
    const int nib = 4 * ((token >> 1) + 4 * (token & 1));
    const uint32_t ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)((ws[e] >> nib) & 15u), s, m);
  }
  if (P.vec) {
    Eight<T> v;
    v.set(y);
    v.store(dst);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) store<T>(dst + e, y[e]);
  }
}

template <typename T, bool APPEND>
static int launch_rows(const KvRowsParams& P, int64_t rows, hipStream_t st, const char* what) {
  // any start inside a block: one block more than the tokens fill
  const dim3 grid((unsigned)((P.tokens + 14) / 8), (unsigned)P.c.kv_heads, (unsigned)rows);
  const dim3 block((unsigned)(2 * P.c.head_dim));
#define TT_ROWS(D, G)                                                                                     \
  if (P.c.head_dim == D && P.c.group_size == G) {                                                         \
    if constexpr (APPEND) hipLaunchKernelGGL((kv_append_int4_kernel<T, D, G>), grid, block, 0, st, P);    \
    else hipLaunchKernelGGL((kv_read_int4_kernel<T, D, G>), grid, block, 0, st, P);                       \
    return check_launch(what);                                                                            \
  }
  TT_ROWS(64, 32) TT_ROWS(64, 64) TT_ROWS(128, 32) TT_ROWS(128, 64) TT_ROWS(128, 128) TT_ROWS(256, 32)
  TT_ROWS(256, 64) TT_ROWS(256, 128)
#undef TT_ROWS
  set_error("%s: unsupported head_dim / group_size", what);
  return TT_ERR_UNSUPPORTED;
}

template <bool APPEND>
static int rows_entry(const tt_int4_cache* cache, void* k, int64_t k_row, int64_t k_token, int64_t k_head, void* v,
                      int64_t v_row, int64_t v_token, int64_t v_head, int dtype, const int32_t* starts,
                      const int32_t* counts, int64_t rows, int64_t tokens, void* stream, const char* what) {
  const int rc = check_cache(cache, rows, what);
  if (rc) return rc;
  TT_REQUIRE(tokens >= 0 && tokens < (1LL << 30), "%s: bad token count", what);
  TT_REQUIRE(valid_out_dtype(dtype), "%s: dtype must be fp16, bf16 or fp32", what);
  if (rows == 0 || tokens == 0) return TT_OK;
  TT_REQUIRE(k && v && starts, "%s: null pointer", what);
  KvRowsParams P{};
  P.c = *cache;
  P.x[0] = k; P.x[1] = v;
  P.x_row[0] = k_row; P.x_row[1] = v_row;
  P.x_token[0] = k_token; P.x_token[1] = v_token;
  P.x_head[0] = k_head; P.x_head[1] = v_head;
  P.starts = starts; P.counts = counts; P.tokens = (int)tokens;
  const int64_t whole = dtype == TT_F32 ? 4 : 8;
  P.vec = aligned(k, 16) && aligned(v, 16) &&
          ((k_row | k_token | k_head | v_row | v_token | v_head) & (whole - 1)) == 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TT_F16) return launch_rows<f16_t, APPEND>(P, rows, st, what);
  if (dtype == TT_BF16) return launch_rows<bf16_t, APPEND>(P, rows, st, what);
  return launch_rows<float, APPEND>(P, rows, st, what);
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_int4_cache_size(void) { return (int64_t)sizeof(tt_int4_cache); }

extern "C" int tt_kv_append_int4(const tt_int4_cache* cache, const void* k, int64_t k_row, int64_t k_token, int64_t k_head,
                                 const void* v, int64_t v_row, int64_t v_token, int64_t v_head, int dtype,
                                 const int32_t* starts, const int32_t* counts, int64_t rows, int64_t tokens,
                                 void* stream) {
  return rows_entry<true>(cache, const_cast<void*>(k), k_row, k_token, k_head, const_cast<void*>(v), v_row, v_token, v_head,
                          dtype, starts, counts, rows, tokens, stream, "kv_append_int4");
}

extern "C" int tt_kv_read_int4(const tt_int4_cache* cache, void* k_out, int64_t k_row, int64_t k_token, int64_t k_head,
                               void* v_out, int64_t v_row, int64_t v_token, int64_t v_head, int dtype,
                               const int32_t* starts, const int32_t* counts, int64_t rows, int64_t tokens, void* stream) {
  return rows_entry<false>(cache, k_out, k_row, k_token, k_head, v_out, v_row, v_token, v_head, dtype, starts, counts, rows,
                           tokens, stream, "kv_read_int4");
}
