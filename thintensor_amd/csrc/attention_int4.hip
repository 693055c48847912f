// Decode attention over the 4-bit KV cache (tt_int4_cache in thintensor_hip.h), one query token per
// sequence, with a window and first tokens, on the 16-bit matrix cores.
//
// A stored value is c s + m with s of seven significant bits, so f16(c s) is exact and
//   q.k_t  = sum_d q_d (c s)_td + sum_groups m_tg (sum of q over the group),
//   out_d  = sum_t p_t (c s)_td + sum_t p_t m_tg
// are products of exact f16 operands added in binary32 (v_mfma_f32_16x16x32_f16):
//   * q is scaled by a power of two per head (its largest element to [2^7, 2^8)), which rounds only
//     what lies 2^-31 below that element; a group's sum of q goes in as three f16 parts;
//   * p is split into an f16 and the f16 of what that leaves, so a weight is off by 2^-21 of itself or
//     2^-31 of the largest; the two sums of an output are rounded each, by 2^-24 of a group's range.
// Scores come out as rows = tokens, columns = query heads: a lane holds eight consecutive tokens of
// one head, which is the operand that the product with V takes, so p never leaves its registers.  The
// product with V is formed transposed (rows = dims, columns = heads), so that a head's running
// maximum, sum and rescaling stay in its column's lanes as well.
//
// One wave takes 32 tokens at a time for up to sixteen query heads of a KV head; the waves of a
// workgroup take turns and are joined in LDS; a long sequence is split over workgroups that leave
// (m, l, o) for a second kernel.  (Sixteen waves in a workgroup, to keep longer rows in one launch, were
// slower everywhere: 1024 tokens of 8 x 64 8.3 us against 8.3 with four, 575 tokens 7.1 against 6.5.)
//
// 131072 and 98304 tokens of 8 KV heads x 128 with 64 query heads (250 MB) take 48 to 51 us and 4.7 for the
// join: 4.9 to 5.2 TB/s.  A tile of 32 tokens costs a wave about 290 vector instructions, two thirds of them to
// form operands from codes (shift, and-or and one packed fma for two values), and 28 matrix instructions;
// the vector units are busy 74% of the time, the matrix cores 25%.  Short rows are bound by
// their round trips: 575 tokens of 8 x 64 6.0 us (6.1 with the first tile requested after q is used), of which
// a launch and one tile are 3.8.
#include "kv_int4.h"
#include "tt_common.h"

namespace tt {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;          // tokens per step of a wave
constexpr int kHeadBlock = 16;     // query heads per workgroup
constexpr int kWaves = 4;
constexpr int kMostSplits = 512;
constexpr int kLongTiles = 256;
// Weights are 2^7 exp(s - m), where m follows the running maximum only when that is more than 2^8 past it:
// they stay below 2^15.
constexpr float kPScale = 7.0f;
constexpr float kSlack = 8.0f;

struct Attn4Params {
  tt_int4_cache c;
  const void* q;
  int64_t q_row, q_head;
  const int32_t* lengths;
  const void* sinks;
  int sink_dtype, q_bf16, q_vec;      // q_vec: rows of q start on 16-byte boundaries
  int heads, per_kv, head_blocks, splits;
  int fill, long_tiles;            // rows that may be long: see Attn4Plan
  int window, first, max_length;
  float scale_log2;                // scale * log2(e)
  float* part_o;                   // [rows, heads, splits, D]
  float2* part_ml;                 // [rows, heads, splits]: (m, l)
  void* out;
  int64_t out_row, out_head;
};

// The visible 32-token tiles of a row: [0, a) and [b, e); tile i of them.
struct Visible {
  int n, start, a, b, e;
  __device__ Visible(const Attn4Params& P, int row) {
    n = min(max(P.lengths[row], 0), P.max_length);
    start = P.window > 0 ? max(0, n - P.window) : 0;
    e = (n + kTile - 1) / kTile;
    b = start / kTile;
    a = min((min(P.first, n) + kTile - 1) / kTile, b);
  }
  __device__ int tiles() const { return a + e - b; }
  __device__ int tile(int i) const { return i < a ? i : b + i - a; }
  // the tiles of a workgroup, while there are some
  __device__ int share(const Attn4Params& P) const {
    const int t = tiles(), even = max(kWaves, (t + P.splits - 1) / P.splits);
    return P.long_tiles == 0 ? even : max(even, min(P.long_tiles, (t + P.fill - 1) / P.fill));
  }
};

// (__builtin_bit_cast of a vector's element takes element 0: a value of its own, always)
__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t pack_h2(float a, float b) { return f32_to_f16_bits(a) | ((uint32_t)f32_to_f16_bits(b) << 16); }

// Eight codes as f16(c s), exactly: register p holds nibbles p and p + 4 (times s[p]).  The nibble goes
// to the top of the mantissa of 16, which makes 16 + c, and one packed fma takes c s from it (off = -16 s;
// steps are at most 4064, so that it is finite).  `mask` sits in a register of its own: an instruction
// takes one constant.
__device__ __forceinline__ h8_t scaled_codes(uint32_t w, const h2 s[4], const h2 off[4], uint32_t mask) {
  const uint32_t x[4] = {w << 6, w << 2, w >> 2, w >> 6};
  u4_t r;
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const uint32_t v = (x[p] & mask) | 0x4c004c00u;
    const h2 c = __builtin_elementwise_fma(as_h2(v), s[p], off[p]);
    r[p] = __builtin_bit_cast(uint32_t, c);
  }
  return __builtin_bit_cast(h8_t, r);
}

// Orders this wave's LDS accesses for its other lanes: a wave's LDS operations execute in order, the
// compiler has to keep them so.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

__device__ __forceinline__ float col_max(float v) {   // over the four lanes of a column
  v = fmaxf(v, xor_partner<16>(v));
  return fmaxf(v, xor_partner<32>(v));
}
__device__ __forceinline__ float col_sum(float v) { return bfly<32>(bfly<16>(v)); }

__device__ __forceinline__ float sink_log2(const Attn4Params& P, int h) {
  const float v = P.sink_dtype == TT_F32    ? reinterpret_cast<const float*>(P.sinks)[h]
                  : P.sink_dtype == TT_BF16 ? to_f32(reinterpret_cast<const bf16_t*>(P.sinks)[h])
                                            : to_f32(reinterpret_cast<const f16_t*>(P.sinks)[h]);
  return v * 0x1.715476p+0f;
}

__device__ __forceinline__ void store_out(const Attn4Params& P, int row, int h, int d, float v) {
  const int64_t at = row * P.out_row + h * P.out_head + d;
  if (P.q_bf16) store<bf16_t>(reinterpret_cast<bf16_t*>(P.out) + at, v);
  else store<f16_t>(reinterpret_cast<f16_t*>(P.out) + at, v);
}

// o / (l + sink), where l and o carry the maximum M; a row that saw nothing is 0.
__device__ __forceinline__ float finish(const Attn4Params& P, int h, float o, float l, float M, bool any) {
  if (!any) return 0.0f;
  if (P.sinks) {
    const float sk = sink_log2(P, h);
    const float top = fmaxf(M, sk);
    const float e = __builtin_amdgcn_exp2f(M - top);
    return o * e / (l * e + __builtin_amdgcn_exp2f(sk - top + kPScale));
  }
  return o / l;
}

// What a wave needs of 32 tokens, in registers: K rows of its lane's token in both halves (its quarter
// of the dims) with their steps and minima, V words of its lane's block of eight tokens with theirs.
template <int D, int G>
struct Tile {
  static constexpr int KW = D / 32, VJ = D / 64;
  static constexpr int LG = D / 4 > G ? D / 4 / G : 1;   // groups in a quarter (1 or 2)
  uint32_t kw[2][KW], ks[2][LG];
  u4_t vw[VJ], vs[VJ], vm;
  static constexpr int NG = D / G;
  // byte offsets of this lane in a tile, beside the tile's own address, which is the wave's
  uint32_t k_at, ks_at, v_at, vs_at, vm_at;
  __device__ __forceinline__ void place(int n, int quad) {
    const int t = 8 * (n >> 2) + (n & 3);          // its token in the first half; four later in the second
    k_at = (uint32_t)(t * (D / 2) + quad * (D / 8));
    ks_at = (uint32_t)(t * (4 * NG) + quad * (D / 4) / G * 4);
    v_at = (uint32_t)(quad * (4 * D) + 16 * n);
    vs_at = (uint32_t)((quad * NG + (G == 32 ? n >> 3 : 0)) * 32);
    // rows past the groups repeat the last one; their products are not used
    vm_at = (uint32_t)((quad * NG + (n < NG ? n : NG - 1)) * 32 + 16);
  }
  __device__ __forceinline__ void load_k(const char* kc, const char* ksp, int t0) {
    const char* k = kc + (int64_t)t0 * (D / 2);
    const char* s = ksp + (int64_t)t0 * (4 * NG);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const char* p = k + (size_t)(k_at + h * (2 * D));
      if constexpr (KW == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        kw[h][0] = v.x; kw[h][1] = v.y;
      } else {
#pragma unroll
        for (int x = 0; x < KW / 4; x++) {
          const u4_t v = *reinterpret_cast<const u4_t*>(p + 16 * x);
#pragma unroll
          for (int e = 0; e < 4; e++) kw[h][4 * x + e] = v[e];
        }
      }
      const char* q = s + (size_t)(ks_at + h * (16 * NG));
      if constexpr (LG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(q);
        ks[h][0] = v.x; ks[h][1] = v.y;
      } else {
        ks[h][0] = *reinterpret_cast<const uint32_t*>(q);
      }
    }
  }
  __device__ __forceinline__ void load_v(const char* vc, const char* vsp, int t0) {
    const char* v = vc + (int64_t)t0 * (D / 2);
    const char* s = vsp + (int64_t)t0 * (4 * NG);
#pragma unroll
    for (int j = 0; j < VJ; j++) {
      vw[j] = *reinterpret_cast<const u4_t*>(v + (size_t)(v_at + j * 256));
      vs[j] = *reinterpret_cast<const u4_t*>(s + (size_t)(vs_at + 64 * j / G * 32));
    }
    vm = *reinterpret_cast<const u4_t*>(s + (size_t)vm_at);
  }
};

template <typename T, int D, int G>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 256 ? 2 : 3))) void attn4_kernel(Attn4Params P) {
  constexpr int NG = D / G;                    // groups of a token
  constexpr int KW = Tile<D, G>::KW, LG = Tile<D, G>::LG;
  constexpr int VT = D / 16;                   // tiles of 16 dims
  constexpr int VJ = D / 64;
  constexpr int OS = D + 4;                    // LDS row of a head
  // Splits next to each other, or last, where short rows have no use for most of them: every row's first one
  // starts before those, and a row's splits are dealt over the CUs (a multiple of 32 apart they would share one).
  int split = blockIdx.x, group = blockIdx.y, row = blockIdx.z;
  if (P.long_tiles != 0) {
    split = blockIdx.z;
    group = blockIdx.x;
    row = __builtin_amdgcn_readfirstlane((int)((blockIdx.y + 5u * blockIdx.z) % gridDim.y));
  }
  const int kvh = group / P.head_blocks, hb = group % P.head_blocks;
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int h0 = kvh * P.per_kv + hb * kHeadBlock;
  const int heads = min(kHeadBlock, P.per_kv - hb * kHeadBlock);
  __shared__ __attribute__((aligned(16))) float o_s[kWaves][16][OS];
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];

  // q is requested before the row's length is known, the first tile before q is used.
  // Element e of step i is dim quad D/4 + 8 i + (e/2) + 4 (e%2)
  const int hq = h0 + min(n, heads - 1);
  uint32_t qw[KW * 4];                         // pairs of elements as they are stored
  {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(P.q) + row * P.q_row + hq * P.q_head + quad * (D / 4);
    if (P.q_vec) {
#pragma unroll
      for (int i = 0; i < KW; i++) {
        const u4_t v = reinterpret_cast<const u4_t*>(q)[i];
#pragma unroll
        for (int e = 0; e < 4; e++) qw[4 * i + e] = v[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < KW * 4; i++) qw[i] = q[2 * i] | ((uint32_t)q[2 * i + 1] << 16);
    }
  }
  const Visible vis(P, row);
  const int nt = vis.tiles(), share = vis.share(P);
  const int first_tile = split * share;
  if (first_tile >= nt && !(nt == 0 && split == 0)) return;
  const int end_tile = min(first_tile + share, nt);

  const char* kc = reinterpret_cast<const char*>(P.c.k_codes) + 4 * (row * P.c.kc_seq + kvh * P.c.kc_head);
  const char* ks = reinterpret_cast<const char*>(P.c.k_scales) + 2 * (row * P.c.ks_seq + kvh * P.c.ks_head);
  const char* vc = reinterpret_cast<const char*>(P.c.v_codes) + 4 * (row * P.c.vc_seq + kvh * P.c.vc_head);
  const char* vs = reinterpret_cast<const char*>(P.c.v_scales) + 2 * (row * P.c.vs_seq + kvh * P.c.vs_head);
  Tile<D, G> tile;
  tile.place(n, quad);
  // (a wave without a tile, of a row without one too, requests one that the cache has: a wait for q behind a
  // branch would wait for the tile as well)
  int i = first_tile + wave, t0 = vis.tile(max(min(i, end_tile - 1), 0)) * kTile;
  tile.load_k(kc, ks, t0);
  tile.load_v(vc, vs, t0);

  // ---- q as f16 operands
  auto qf = [&](int i) __attribute__((always_inline)) {
    return (i & 1) ? hi_f32<T>(qw[i / 2]) : lo_f32<T>(qw[i / 2]);
  };
  float big = 0.0f, poison = 0.0f;
#pragma unroll
  for (int i = 0; i < KW * 8; i++) {
    const float v = qf(i);
    big = fmaxf(big, __builtin_fabsf(v));
    poison += v * 0.0f;
  }
  big = col_max(big);
  poison = col_sum(poison);
  // the exponent of the largest element, limited so that both powers of two are normal
  int ex = (int)(__builtin_bit_cast(uint32_t, big) >> 23) - 127 - 7;
  if (ex < -110) ex = -110;
  // the sign of the scale goes to q, so that the largest product is the largest score
  float down = poison == poison ? pow2i(-ex) : poison;
  if (P.scale_log2 < 0.0f) down = -down;
  const float score_scale = fmaxf(__builtin_fabsf(P.scale_log2) * pow2i(ex), 0x1p-126f);
  h8_t qb[KW], qm;
  {
    float part[LG];
#pragma unroll
    for (int j = 0; j < LG; j++) part[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < KW; i++) {
      u4_t r;
#pragma unroll
      for (int p = 0; p < 4; p++) r[p] = pack_h2(qf(8 * i + p) * down, qf(8 * i + p + 4) * down);
      qb[i] = __builtin_bit_cast(h8_t, r);
#pragma unroll
      for (int e = 0; e < 8; e++) part[i * LG / KW] += (float)qb[i][e];
    }
    uint16_t limb[6] = {0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < LG; j++)
#pragma unroll
      for (int k = 0; k < 3; k++) {
        limb[3 * j + k] = f32_to_f16_bits(part[j]);
        part[j] -= to_f32(f16_t{limb[3 * j + k]});
      }
    const u4_t r = {limb[0] | ((uint32_t)limb[1] << 16), limb[2] | ((uint32_t)limb[3] << 16), limb[4] | ((uint32_t)limb[5] << 16), 0u};
    qm = __builtin_bit_cast(h8_t, r);
  }

  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  f4_t o[VT], om = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < VT; i++) o[i] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
  float m_run = ninf, l_run = 0.0f;

  uint32_t mask = 0x03c003c0u;
  asm volatile("" : "+v"(mask));

  auto step = [&](int t0, int next) __attribute__((always_inline)) {
    // ---- scores: register e of half h is token t0 + 8 quad + 4 h + e of head n
    f4_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      sc[h] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
      const uint32_t ma = tile.ks[h][0] >> 16, mb = LG > 1 ? tile.ks[h][LG - 1] >> 16 : 0u;
      const u4_t r = {ma | (ma << 16), ma | (mb << 16), mb | (mb << 16), 0u};
      sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, r), qm, sc[h], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < LG; j++) {
        const h2 sm = as_h2(tile.ks[h][j]);
        const h2 s1 = {sm[0], sm[0]};
        const h2 o1 = s1 * (h2){(_Float16)-16.0f, (_Float16)-16.0f};
        const h2 s4[4] = {s1, s1, s1, s1}, o4[4] = {o1, o1, o1, o1};
#pragma unroll
        for (int x = j * KW / LG; x < (j + 1) * KW / LG; x++)
          sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(scaled_codes(tile.kw[h][x], s4, o4, mask), qb[x], sc[h], 0, 0, 0);
      }
    }
    tile.load_k(kc, ks, next);
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) s[e] = sc[e >> 2][e & 3];
    const bool whole = t0 + kTile <= vis.n && (t0 >= vis.start || t0 + kTile <= P.first);
    if (!whole) {
      // tokens out of sight: no score, and V's step and minimum 0 (what lies there may be NaN)
      uint32_t keep[4];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int t = t0 + 8 * quad + e;
        const bool in = t < vis.n && (t >= vis.start || t < P.first);
        if (!in) s[e] = ninf;
        if ((e & 1) == 0) keep[e >> 1] = in ? 0xffffu : 0u;
        else keep[e >> 1] |= in ? 0xffff0000u : 0u;
      }
#pragma unroll
      for (int p = 0; p < 4; p++) {
        tile.vm[p] &= keep[p];
#pragma unroll
        for (int j = 0; j < VJ; j++) tile.vs[j][p] &= keep[p];
      }
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
    // no lane of a column past its maximum by more than the slack: nothing moves
    if (__builtin_amdgcn_ballot_w64(top * score_scale > m_run + kSlack) != 0) {
      const float m_new = fmaxf(m_run, col_max(top) * score_scale);
      const float a = m_new == ninf ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= a;
#pragma unroll
      for (int x = 0; x < VT; x++) o[x] *= a;
      om *= a;
      m_run = m_new;
    }
    const float base = kPScale - (m_run == ninf ? 0.0f : m_run);
    u4_t hi, lo;
#pragma unroll
    for (int p = 0; p < 4; p++) {
      const float pa = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p], score_scale, base));
      const float pb = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p + 1], score_scale, base));
      l_run += pa + pb;
      // both parts towards zero: the second one takes what the first leaves
      const uint32_t hw = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(pa, pb));
      const h2 hh = as_h2(hw);
      hi[p] = hw;
      lo[p] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)hh[0], -1.0f, pa), __builtin_fmaf((float)hh[1], -1.0f, pb)));
    }
    const h8_t ph = __builtin_bit_cast(h8_t, hi), pl = __builtin_bit_cast(h8_t, lo);

    // ---- values: register r of o[4 j + x] is dim 64 j + 4 (4 quad + r) + x of head n
    const h8_t vmh = __builtin_bit_cast(h8_t, tile.vm);   // rows = groups
    om = __builtin_amdgcn_mfma_f32_16x16x32_f16(vmh, ph, om, 0, 0, 0);
    om = __builtin_amdgcn_mfma_f32_16x16x32_f16(vmh, pl, om, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < VJ; j++) {
      const h2 s4[4] = {as_h2(tile.vs[j][0]), as_h2(tile.vs[j][1]), as_h2(tile.vs[j][2]), as_h2(tile.vs[j][3])};
      h2 o4[4];
#pragma unroll
      for (int p = 0; p < 4; p++) o4[p] = s4[p] * (h2){(_Float16)-16.0f, (_Float16)-16.0f};
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const h8_t v = scaled_codes(tile.vw[j][x], s4, o4, mask);
        o[4 * j + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[4 * j + x], 0, 0, 0);
        o[4 * j + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[4 * j + x], 0, 0, 0);
      }
    }
    tile.load_v(vc, vs, next);
  };

  // K of the next tile is requested as soon as the scores have taken the present one's, V after the
  // products with it (past the end: the last tile once more)
  for (; i < end_tile; i += kWaves) {
    const int next = vis.tile(min(i + kWaves, end_tile - 1)) * kTile;
    step(t0, next);
    t0 = next;
  }

  // ---- join the waves.  The groups' sums of p m sit in the column's lanes of quads 0 and 1.
  const float l_col = col_sum(l_run);
  {
    float* mine = o_s[wave][n];
    if (4 * quad < NG) {   // staged through the row, read back by its four lanes below
#pragma unroll
      for (int r = 0; r < 4; r++) mine[4 * quad + r] = om[r];
    }
    wave_lds_fence();
    float gm[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) gm[g] = mine[g];
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < VJ; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = 64 * j + 16 * quad + 4 * r;
        float add = gm[0];
#pragma unroll
        for (int g = 1; g < NG; g++) add = d / G == g ? gm[g] : add;
        f4_t v;
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = o[4 * j + x][r] + add;
        *reinterpret_cast<f4_t*>(mine + d) = v;
      }
    if (quad == 0) {
      m_s[wave][n] = m_run;
      l_s[wave][n] = l_col;
    }
  }
  __syncthreads();
  const bool only = nt <= share;
  for (int u = threadIdx.x; u < heads * D; u += 64 * kWaves) {
    const int hh = u / D, d = u % D;
    float M = m_s[0][hh];
#pragma unroll
    for (int w = 1; w < kWaves; w++) M = fmaxf(M, m_s[w][hh]);
    const float base = M == ninf ? 0.0f : M;
    float acc = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float e = __builtin_amdgcn_exp2f(m_s[w][hh] - base);
      acc = __builtin_fmaf(o_s[w][hh][d], e, acc);
      l = __builtin_fmaf(l_s[w][hh], e, l);
    }
    if (only) {
      store_out(P, row, h0 + hh, d, finish(P, h0 + hh, acc, l, M, nt > 0));
    } else {
      const int64_t at = ((int64_t)row * P.heads + h0 + hh) * P.splits + split;
      P.part_o[at * D + d] = acc;
      if (d == 0) P.part_ml[at] = make_float2(M, l);
    }
  }
}

// Joins the splits of one (row, head), two or more; rows that one workgroup finished are left alone.
// 32 splits of 128 (row, head) x 128 take 4.8 us, mostly the launch and two round trips (a thread per dim
// that walked over the splits: 33).
// Every wave forms all weights (a split per lane); sixteen bytes of a split's o per thread, the splits
// dealt over the threads' rows and joined in LDS.
// One wave where there are more than four (row, head) for each CU, which fill the chip by themselves: 4096 without a join
// 3.9 us, 8.7 with 256 threads.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void attn4_fold_kernel(Attn4Params P) {
  constexpr int PIECES = D / 4, ROWS = THREADS / PIECES;
  const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63;
  const int piece = threadIdx.x % PIECES, r = threadIdx.x / PIECES;
  __shared__ float e_s[kMostSplits];
  __shared__ __attribute__((aligned(16))) f4_t sum[ROWS][PIECES];
  const int64_t at = ((int64_t)row * P.heads + h) * P.splits;
  const float2* ml = P.part_ml + at;
  const f4_t* po = reinterpret_cast<const f4_t*>(P.part_o + at * D);
  // requested before the row's length is known, all inside the scratch: what no workgroup wrote is not used
  constexpr int PRE = 4;
  float2 first = ml[min(lane, P.splits - 1)];
  f4_t pre[PRE];
#pragma unroll
  for (int k = 0; k < PRE; k++) pre[k] = po[(int64_t)min(r + k * ROWS, P.splits - 1) * PIECES + piece];
  const Visible vis(P, row);
  const int nt = vis.tiles(), share = vis.share(P);
  if (nt <= share) return;
  const int parts = (nt + share - 1) / share;
  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  if (lane >= parts) first = make_float2(ninf, 0.0f);
  float M = first.x;
  for (int k = lane + 64; k < parts; k += 64) M = fmaxf(M, ml[k].x);
#define TT_LEVEL(X) M = fmaxf(M, xor_partner<X>(M));
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
  const float base = M == ninf ? 0.0f : M;
  float l = 0.0f;
  for (int k = lane; k < parts; k += 64) {
    const float2 v = k == lane ? first : ml[k];
    const float e = __builtin_amdgcn_exp2f(v.x - base);
    l = __builtin_fmaf(v.y, e, l);
    if (threadIdx.x < 64) e_s[k] = e;
  }
  l = xor_sum(l, 1, 64);
  __syncthreads();
  f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < PRE; k++)
    if (r + k * ROWS < parts) acc += pre[k] * e_s[r + k * ROWS];
  constexpr int MORE = 16;              // (past the end: the last one, weight 0)
  for (int i = r + PRE * ROWS; i < parts; i += MORE * ROWS) {
    f4_t more[MORE];
#pragma unroll
    for (int k = 0; k < MORE; k++) more[k] = po[(int64_t)min(i + k * ROWS, parts - 1) * PIECES + piece];
#pragma unroll
    for (int k = 0; k < MORE; k++) acc += more[k] * (i + k * ROWS < parts ? e_s[i + k * ROWS] : 0.0f);
  }
  sum[r][piece] = acc;
  __syncthreads();
  if (r == 0) {
#pragma unroll
    for (int k = 1; k < ROWS; k++) acc += sum[k][piece];
#pragma unroll
    for (int x = 0; x < 4; x++) store_out(P, row, h, 4 * piece + x, finish(P, h, acc[x], l, M, true));
  }
}

// Tiles that a row may see at most, and the workgroups that share them.
static int64_t most_tiles(int64_t limit, int64_t window, int64_t first) {
  const int64_t all = (limit + kTile - 1) / kTile;
  if (window <= 0) return all;
  const int64_t some = (first + kTile - 1) / kTile + (window + kTile - 1) / kTile + 1;
  return some < all ? some : all;
}

struct Attn4Plan {
  int64_t limit, window, first, head_blocks, splits;
  int64_t fill, long_tiles;   // 0, or what bounds a workgroup's tiles beside `splits`: see split_rows
};

// Workgroups that share a row: few tiles are taken by one, since a second launch has to join several
// (8 groups of sequence and KV head, head_dim 64: 19 tiles 6.6 us by one and 8.0 shared, 32 tiles 8.3 and
// 7.8, 64 tiles 13.4 and 7.9), and more of them while there are groups for the chip (256 groups, one for each CU:
// 16 tiles 6.5 and 10.4, 64 tiles 13.9 and 16.0).  Shared, up to two workgroups for each CU, 512, and eight tiles
// each: 16384 tokens of 8 x 64, 1024 workgroups 11.7 us, 512 9.8; 52428 tokens of 2 x 10 x 128, 520
// workgroups, of which some CUs take a third one, 43.0, 500 33.0.
// Lengths are not known here.  So that one long row among short ones is not left to a few workgroups, none takes
// more than kLongTiles tiles; of the splits that this adds a row uses what the chip has room for, or its length
// needs (64 rows of 8 KV heads x 128, capacity 65536: one row of 65536 among 500s 94 us, 383 without; all of 500
// 18.5 and 13.6, of 16384 228 and 215, lengths up to 16384 138 and 149; of 512 tiles 113, 17.2, 226 and 154).
static void split_rows(int64_t groups, int64_t tiles, Attn4Plan* p) {
  const int64_t cus = device_cus();
  p->splits = 1;
  p->long_tiles = 0;
  p->fill = groups < 2 * cus ? 2 * cus / groups : 1;
  if (tiles <= 24 || (groups >= cus && tiles <= 64)) return;
  const int64_t most = (tiles + 7) / 8, s = p->fill < most ? p->fill : most;
  const int64_t for_long = (tiles + kLongTiles - 1) / kLongTiles;
  p->splits = s > for_long ? s : for_long;
  if (p->splits > s) p->long_tiles = kLongTiles;
  if (p->splits > kMostSplits) p->splits = kMostSplits;
}

static Attn4Plan plan(const tt_int4_cache* c, int64_t rows, int64_t heads, int64_t window, int64_t first, int64_t max_length) {
  Attn4Plan p;
  p.limit = max_length < c->capacity ? max_length : c->capacity;
  p.window = window > p.limit ? 0 : (window > 0 ? window : 0);
  p.first = p.window == 0 ? 0 : (first < p.limit ? first : p.limit);
  p.head_blocks = (heads / c->kv_heads + kHeadBlock - 1) / kHeadBlock;
  split_rows(rows * c->kv_heads * p.head_blocks, most_tiles(p.limit, p.window, p.first), &p);
  return p;
}

template <int D, int G>
static int launch_attn4(const Attn4Params& P, int64_t rows, hipStream_t st, const char* what) {
  const unsigned groups = (unsigned)(P.c.kv_heads * P.head_blocks);
  const dim3 grid = P.long_tiles ? dim3(groups, (unsigned)rows, (unsigned)P.splits) : dim3((unsigned)P.splits, groups, (unsigned)rows);
  if (P.q_bf16) hipLaunchKernelGGL((attn4_kernel<bf16_t, D, G>), grid, dim3(64 * kWaves), 0, st, P);
  else hipLaunchKernelGGL((attn4_kernel<f16_t, D, G>), grid, dim3(64 * kWaves), 0, st, P);
  const int rc = check_launch(what);
  if (rc || P.splits == 1) return rc;
  const dim3 pairs((unsigned)P.heads, (unsigned)rows);
  if (P.heads * rows > 4 * device_cus()) hipLaunchKernelGGL((attn4_fold_kernel<D, 64>), pairs, dim3(64), 0, st, P);
  else hipLaunchKernelGGL((attn4_fold_kernel<D, 256>), pairs, dim3(256), 0, st, P);
  return check_launch(what);
}

static int check_attention(const tt_int4_cache* c, int64_t rows, int64_t heads, int64_t window, int64_t first,
                           int64_t max_length, const char* what) {
  const int rc = check_cache(c, rows, what);
  if (rc) return rc;
  TT_REQUIRE(heads > 0 && heads % c->kv_heads == 0, "%s: heads must be a multiple of kv_heads", what);
  TT_REQUIRE(heads <= 65535 && c->kv_heads * ((heads / c->kv_heads + kHeadBlock - 1) / kHeadBlock) <= 65535, "%s: too many heads", what);
  TT_REQUIRE(window >= 0 && first >= 0 && max_length > 0, "%s: window, first_tokens and max_length must not be negative (max_length at least 1)", what);
  return TT_OK;
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_gqa_attention_int4_scratch_floats(const tt_int4_cache* cache, int64_t rows, int64_t heads,
                                                        int64_t window, int64_t first_tokens, int64_t max_length) {
  if (check_attention(cache, rows, heads, window, first_tokens, max_length, "gqa_attention_int4") != TT_OK) return TT_ERR_INVALID;
  if (rows == 0) return 0;
  const Attn4Plan p = plan(cache, rows, heads, window, first_tokens, max_length);
  return p.splits == 1 ? 0 : rows * heads * p.splits * (cache->head_dim + 2);
}

extern "C" int tt_gqa_attention_int4(const tt_int4_cache* cache, const void* q, int64_t q_row, int64_t q_head, int dtype,
                                     const int32_t* lengths, int64_t rows, int64_t heads, int64_t window,
                                     int64_t first_tokens, int64_t max_length, const void* sinks, int sink_dtype,
                                     float scale, float* scratch, int64_t scratch_floats, void* out, int64_t out_row,
                                     int64_t out_head, void* stream) {
  const char* what = "gqa_attention_int4";
  const int rc = check_attention(cache, rows, heads, window, first_tokens, max_length, what);
  if (rc) return rc;
  TT_REQUIRE(valid_act_dtype(dtype), "%s: q must be fp16 or bf16", what);
  TT_REQUIRE(sinks == nullptr || valid_out_dtype(sink_dtype), "%s: sinks must be fp16, bf16 or fp32", what);
  TT_REQUIRE(scale - scale == 0.0f, "%s: scale must be finite", what);
  if (rows == 0) return TT_OK;
  TT_REQUIRE(q && out && lengths, "%s: null pointer", what);
  // every output has one writer; in place each workgroup reads its own heads of q before it writes them
  const Region qr(q, 2, cache->head_dim, {{rows, q_row}, {heads, q_head}});
  const Region made(out, 2, cache->head_dim, {{rows, out_row}, {heads, out_head}});
  TT_REQUIRE(made.once() && (made.same(qr) || apart(made, qr)) && CacheRegions(cache, rows).apart_from(made),
             "%s: out may be q, but must not share memory with itself, the cache or q otherwise", what);
  const Attn4Plan p = plan(cache, rows, heads, window, first_tokens, max_length);
  TT_REQUIRE(p.splits == 1 || (scratch && aligned(scratch, 16) && scratch_floats >= rows * heads * p.splits * (cache->head_dim + 2)),
             "%s: scratch too small or not 16-byte aligned", what);
  Attn4Params P{};
  P.c = *cache;
  P.q = q; P.q_row = q_row; P.q_head = q_head; P.q_bf16 = dtype == TT_BF16;
  P.q_vec = aligned(q, 16) && q_row % 8 == 0 && q_head % 8 == 0;
  P.lengths = lengths;
  P.sinks = sinks; P.sink_dtype = sink_dtype;
  P.heads = (int)heads; P.per_kv = (int)(heads / cache->kv_heads);
  P.head_blocks = (int)p.head_blocks; P.splits = (int)p.splits; P.fill = (int)p.fill; P.long_tiles = (int)p.long_tiles;
  P.window = (int)p.window; P.first = (int)p.first; P.max_length = (int)p.limit;
  P.scale_log2 = (float)((double)scale * 1.4426950408889634);
  P.part_o = scratch;
  P.part_ml = reinterpret_cast<float2*>(scratch + rows * heads * p.splits * cache->head_dim);
  P.out = out; P.out_row = out_row; P.out_head = out_head;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define TT_ATTN4(D, G) \
  if (cache->head_dim == D && cache->group_size == G) return launch_attn4<D, G>(P, rows, st, what);
  TT_ATTN4(64, 32) TT_ATTN4(64, 64) TT_ATTN4(128, 32) TT_ATTN4(128, 64) TT_ATTN4(128, 128) TT_ATTN4(256, 32)
  TT_ATTN4(256, 64) TT_ATTN4(256, 128)
#undef TT_ATTN4
  set_error("%s: unsupported head_dim / group_size", what);
  return TT_ERR_UNSUPPORTED;
}
