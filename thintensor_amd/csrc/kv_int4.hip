// Packing tokens into the 4-bit KV cache and reading them back (layout and rounding: tt_int4_cache
// and tt_kv_append_int4 in thintensor_hip.h).
//
// A workgroup owns whole blocks of eight cache tokens of one sequence and KV head: the V words hold
// eight tokens, so a word has one writer, which merges the tokens it was not given from memory.  Half
// of its threads pack K, half V, two blocks at a time; a thread holds sixteen dims of one token, and a
// group's extremes are exact under any order, taken over its 2, 4 or 8 lanes.
//
// Packing 16384 tokens of 8 KV heads x 128 (85 MB with what is written) takes 24 us, 3.5 TB/s (28 where the inputs
// come from memory): vector instructions, 18 a value, hold 60% of the time, the rest are round trips to memory.  (One block per
// workgroup and eight dims per thread: 38; several blocks and codes decided in binary64 without branches:
// 30, eight dims, 24, sixteen.)  Reading them back takes 16.6 us, 5.1 TB/s, of which four fifths are
// written (an earlier form took 20, with one block requested at a time 23, with heads as the fastest grid axis 22).
#include "kv_int4.h"
#include "tt_common.h"
#include "tt_eight.h"

namespace tt {

constexpr int kMostBlocks = 8;
constexpr int kAhead = 4;

struct KvRowsParams {
  tt_int4_cache c;
  void* x[2];              // k, v
  int64_t x_row[2], x_token[2], x_head[2];
  const int32_t* starts;
  const int32_t* counts;
  int blocks_per;          // blocks of eight cache tokens that a workgroup takes
  int tokens, vec;         // vec: eight elements of k and v start on 16-byte boundaries
};

// A group's step, and codes, are decided in binary64, which costs what binary32 does here and where hi - m and
// x - m are exact (their operands within 2^28 of each other, always so for fp16) and decide ties.

// The smallest s of seven significant bits with 15 s >= hi - m; the product with 1/15 only proposes it.
__device__ __forceinline__ double group_step(float hi, float m) {
  const double reach = (double)hi - (double)m;
  const double raw = reach * (1.0 / 15.0);
  int e = (int)((__builtin_bit_cast(uint64_t, raw) >> 52) & 2047) - 1022 - 7;   // lsb of 7 bits
  if (e < -24) e = -24;
  const double lsb = __builtin_amdgcn_ldexp(1.0, e);
  double s = __builtin_ceil(__builtin_amdgcn_ldexp(raw, -e)) * lsb;
  if (15.0 * (s - lsb) >= reach) s -= lsb;
  if (15.0 * s < reach) s += lsb;
  return reach > 0.0 ? __builtin_fmin(s, 4064.0) : 0.0;
}

// (x - m) / s to the nearest code, ties to even.  The quotient is corrected by its residual, which
// makes it exact where it has few bits (a tie is j + 1/2) and keeps every other off the ties; 1.5 2^52
// added leaves its nearest integer in the low word.  x is limited to [m, top], top = m + 15 s in binary32:
// no less than the group's maximum, except where s has reached its end and codes past 15 are cut.
__device__ __forceinline__ uint32_t code_of(float x, float m, float top, double md, double s, double inv) {
  const double d = (double)__builtin_amdgcn_fmed3f(x, m, top) - md;
  const double y0 = d * inv;
  const double y = __builtin_fma(__builtin_fma(-y0, s, d), inv, y0);
  return (uint32_t)__builtin_bit_cast(uint64_t, y + 6755399441055744.0);
}

// Extremes of a group over G / 16 neighbouring lanes, as integers in the order of the values.
__device__ __forceinline__ int ordered(float x) {
  const int b = __builtin_bit_cast(int, x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float of_ordered(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }

template <int M> __device__ __forceinline__ int xor_int(int v) {
  return __builtin_bit_cast(int, xor_partner<M>(__builtin_bit_cast(float, v)));
}

template <int G>
__device__ __forceinline__ void group_extremes(int& lo, int& hi) {
#define TT_LEVEL(M)                   \
  if (G / 16 > M) {                   \
    lo = min(lo, xor_int<M>(lo));     \
    hi = max(hi, xor_int<M>(hi));     \
  }
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4)
#undef TT_LEVEL
}

// The cache tokens of this workgroup: blocks of eight from `block` up to `end`, and which of a row's
// tokens lie there.
struct BlockRows {
  int start, count, block, end;
  __device__ BlockRows(const KvRowsParams& P, int row, int part) {
    start = P.starts[row];
    count = P.counts ? min(P.counts[row], P.tokens) : P.tokens;
    // beyond these no token is inside the cache, within them positions fit 32 bits
    if (start >= P.c.capacity || start <= -(1 << 30)) count = 0;
    const int first = (start >> 3) + part * P.blocks_per;
    const int64_t past = min((int64_t)start + max(count, 0) + 7, (int64_t)P.c.capacity) >> 3;
    block = max(first, 0);
    end = (int)min((int64_t)first + P.blocks_per, past);
    if (count <= 0) end = block;
  }
};

template <typename T, int D, int G>
__global__ __launch_bounds__(2 * D) void kv_append_int4_kernel(KvRowsParams P) {
  constexpr int W = D / 16;                        // lanes per token, two words each
  constexpr int NG = D / G;
  __shared__ uint2 vw[2][16][W];
  const int row = blockIdx.z, head = blockIdx.y;
  const BlockRows R(P, row, (int)blockIdx.x);
  if (R.block >= R.end) return;
  const int which = __builtin_amdgcn_readfirstlane((int)threadIdx.x / D);   // 0: K, 1: V; whole waves
  const int tid = (int)threadIdx.x % D;
  const int token = tid / W, word = tid % W;       // of two blocks' sixteen
  const bool first = word % (G / 16) == 0;         // writes the group's scales
  const T* src = reinterpret_cast<const T*>(P.x[which]) + row * P.x_row[which] + head * P.x_head[which] + 16 * word;
  const int64_t x_token = P.x_token[which];
  // this thread's words of a block: of K its token's, of V its dim's
  uint32_t* out = which == 0 ? reinterpret_cast<uint32_t*>(P.c.k_codes) + row * P.c.kc_seq + head * P.c.kc_head + 2 * tid
                             : reinterpret_cast<uint32_t*>(P.c.v_codes) + row * P.c.vc_seq + head * P.c.vc_head + tid;
  uint16_t* scales = which == 0 ? reinterpret_cast<uint16_t*>(P.c.k_scales) + row * P.c.ks_seq + head * P.c.ks_head +
                                      (token * NG + word / (G / 16)) * 2
                                : reinterpret_cast<uint16_t*>(P.c.v_scales) + row * P.c.vs_seq + head * P.c.vs_head +
                                      (token / 8 * NG + word / (G / 16)) * 16 + token % 8;
  Eight<T> next[2];
  auto request = [&](int block) __attribute__((always_inline)) {
    const int t = 8 * block + token - R.start;
    const T* p = src + min(max(t, 0), R.count - 1) * x_token;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (P.vec) {
        next[h].load(p + 8 * h);
      } else {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = to_f32(p[8 * h + e]);
        next[h].set(y);                            // back to what was stored
      }
    }
  };
  request(R.block);
  int buffer = 0;
  for (int block = R.block; block < R.end; block += 2, buffer ^= 1) {
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = next[e >> 3].get(e & 7);
    if (block + 2 < R.end) request(block + 2);
    const int t = 8 * block + token - R.start;
    const bool valid = t >= 0 && t < R.count && block + token / 8 < R.end;
    // extremes; a NaN stays one here and orders past the infinity of its sign
    float lof = x[0], hif = x[0];
#pragma unroll
    for (int e = 1; e < 16; e++) {
      lof = __builtin_elementwise_minimum(lof, x[e]);
      hif = __builtin_elementwise_maximum(hif, x[e]);
    }
    int lo = ordered(lof), hi = ordered(hif);
    group_extremes<G>(lo, hi);
    const bool finite = hi < 0x7f800000 && lo > ordered(__builtin_bit_cast(float, 0xff800000u));
    const float m = round_f16(__builtin_amdgcn_fmed3f(of_ordered(lo), -65504.0f, 65504.0f));
    const double s = finite ? group_step(of_ordered(hi), m) : 0.0;
    const float sf = (float)s;
    uint2 codes = make_uint2(0, 0);
    if (s > 0.0) {
      const double md = (double)m;
      const float top = m + 15.0f * sf;
      double inv = __builtin_amdgcn_rcp(s);
      inv = __builtin_fma(__builtin_fma(-s, inv, 1.0), inv, inv);
      inv = __builtin_fma(__builtin_fma(-s, inv, 1.0), inv, inv);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        codes.x |= code_of(x[e], m, top, md, s, inv) << (4 * e);
        codes.y |= code_of(x[8 + e], m, top, md, s, inv) << (4 * e);
      }
    }
    // a group that is not finite reads as NaN
    const uint32_t mb = finite ? f32_to_f16_bits(m) : 0x7e00u, sb = finite ? f32_to_f16_bits(sf) : 0x7e00u;
    if (which == 0) {
      if (valid) {
        *reinterpret_cast<uint2*>(out + (int64_t)block * D) = codes;
        if (first) *reinterpret_cast<uint32_t*>(scales + (int64_t)block * (16 * NG)) = sb | (mb << 16);
      }
    } else {
      vw[buffer][token][word] = codes;
      if (valid && first) {
        scales[(int64_t)block * (16 * NG)] = (uint16_t)sb;
        scales[(int64_t)block * (16 * NG) + 8] = (uint16_t)mb;
      }
    }
    lds_barrier();                                 // the other buffer's readers are past it as well
    if (which == 1) {
      // this thread's dim of a block's eight tokens; the tokens that were not given keep their codes
      const uint32_t* words = reinterpret_cast<const uint32_t*>(&vw[buffer][0][0]);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (block + h >= R.end) break;
        uint32_t word_out = 0, keep = 0;
#pragma unroll
        for (int k = 0; k < 8; k++)
          word_out |= ((words[(8 * h + k) * (D / 8) + tid / 8] >> (4 * (tid % 8))) & 15u) << (4 * ((k >> 1) + 4 * (k & 1)));
        const int t0 = 8 * (block + h) - R.start;
        if (t0 < 0 || t0 + 8 > R.count) {
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (t0 + k < 0 || t0 + k >= R.count) keep |= 15u << (4 * ((k >> 1) + 4 * (k & 1)));
          word_out = (word_out & ~keep) | (out[(int64_t)(block + h) * D] & keep);
        }
        out[(int64_t)(block + h) * D] = word_out;
      }
    }
  }
}

template <typename T, int D, int G>
__global__ __launch_bounds__(2 * D) void kv_read_int4_kernel(KvRowsParams P) {
  constexpr int W = D / 8;
  constexpr int NG = D / G;
  const int row = blockIdx.z, head = blockIdx.y;
  const BlockRows R(P, row, (int)blockIdx.x);
  if (R.block >= R.end) return;
  const int which = __builtin_amdgcn_readfirstlane((int)threadIdx.x / D);
  const int tid = (int)threadIdx.x % D;
  const int token = tid / W, word = tid % W;
  T* dst = reinterpret_cast<T*>(P.x[which]) + row * P.x_row[which] + head * P.x_head[which] + 8 * word;
  const int64_t x_token = P.x_token[which];
  const uint32_t* codes = which == 0 ? reinterpret_cast<const uint32_t*>(P.c.k_codes) + row * P.c.kc_seq + head * P.c.kc_head + tid
                                     : reinterpret_cast<const uint32_t*>(P.c.v_codes) + row * P.c.vc_seq + head * P.c.vc_head + 8 * word;
  const uint16_t* scales = which == 0 ? reinterpret_cast<const uint16_t*>(P.c.k_scales) + row * P.c.ks_seq + head * P.c.ks_head +
                                            (token * NG + word / (G / 8)) * 2
                                      : reinterpret_cast<const uint16_t*>(P.c.v_scales) + row * P.c.vs_seq + head * P.c.vs_head +
                                            word / (G / 8) * 16 + token;
  const int m_at = which == 0 ? 1 : 8;
  const int nib = 4 * ((token >> 1) + 4 * (token & 1));
  // up to kAhead blocks are requested together, before the first store, which a later load would wait for
  for (int b0 = R.block; b0 < R.end; b0 += kAhead) {
    uint16_t s_bits[kAhead], m_bits[kAhead];
    uint4 w0[kAhead], w1[kAhead];                  // K: the word in w0.x
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const int block = min(b0 + k, R.end - 1);
      const uint32_t* c = codes + (int64_t)block * D;
      s_bits[k] = scales[(int64_t)block * (16 * NG)];
      m_bits[k] = scales[(int64_t)block * (16 * NG) + m_at];
      if (which == 0) {
        w0[k].x = *c;
      } else {
        w0[k] = reinterpret_cast<const uint4*>(c)[0];
        w1[k] = reinterpret_cast<const uint4*>(c)[1];
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const float s = to_f32(f16_t{s_bits[k]}), m = to_f32(f16_t{m_bits[k]});
      float y[8];
      if (which == 0) {
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)((w0[k].x >> (4 * e)) & 15u), s, m);
      } else {
        const uint32_t ws[8] = {w0[k].x, w0[k].y, w0[k].z, w0[k].w, w1[k].x, w1[k].y, w1[k].z, w1[k].w};
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = __builtin_fmaf((float)((ws[e] >> nib) & 15u), s, m);
      }
      const int t = 8 * (b0 + k) + token - R.start;
      if (b0 + k >= R.end || t < 0 || t >= R.count) continue;
      T* o = dst + t * x_token;
      if (P.vec) {
        Eight<T> v;
        v.set(y);
        v.store(o);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) store<T>(o + e, y[e]);
      }
    }
  }
}

template <typename T, bool APPEND>
static int launch_rows(KvRowsParams P, int64_t rows, hipStream_t st, const char* what) {
  // any start inside a block: one block more than the tokens fill
  const int64_t blocks = (P.tokens + 14) / 8;
  // Blocks of a workgroup: as many as leave the chip its fill of workgroups, up to eight (packing is
  // indifferent to half or twice as many; reading 8193 tokens of 10 x 128: 16.6 us with half as many, 14.3,
  // 15.0 with twice as many; one block each at 16384 of 8 x 128: 35 us against 20).
  const int64_t fill = blocks * P.c.kv_heads * rows * P.c.head_dim / (device_cus() * (APPEND ? 2048 : 1024));
  P.blocks_per = (int)(fill < 2 ? (APPEND ? 2 : 1) : fill > kMostBlocks ? kMostBlocks : fill & ~1);
  const dim3 grid((unsigned)((blocks + P.blocks_per - 1) / P.blocks_per), (unsigned)P.c.kv_heads, (unsigned)rows);
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
  TT_REQUIRE(tokens >= 0 && tokens <= (1 << 26), "%s: at most 2^26 tokens of a row", what);
  TT_REQUIRE(valid_out_dtype(dtype), "%s: dtype must be fp16, bf16 or fp32", what);
  if (rows == 0 || tokens == 0) return TT_OK;
  TT_REQUIRE(k && v && starts, "%s: null pointer", what);
  const CacheRegions held(cache, rows);
  if (APPEND) {   // a word of the cache has one writer (reading sequences that share their tokens is fine)
    TT_REQUIRE(held.once(), "%s: sequences, heads and arrays that are written must not share memory", what);
  } else {
    const int64_t element = dtype == TT_F32 ? 4 : 2;
    const Region ko(k, element, cache->head_dim, {{rows, k_row}, {tokens, k_token}, {cache->kv_heads, k_head}});
    const Region vo(v, element, cache->head_dim, {{rows, v_row}, {tokens, v_token}, {cache->kv_heads, v_head}});
    TT_REQUIRE(ko.once() && vo.once() && apart(ko, vo) && held.apart_from(ko) && held.apart_from(vo),
               "%s: outputs must not share memory with themselves, each other or the cache", what);
  }
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
