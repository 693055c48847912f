// Paged attention for few columns (a row's queries of one KV head: single tokens, drafts, short chunks; or a
// small batch against its shared pages): one wave takes 32 tokens at a time for 16 NB columns, the waves of a workgroup
// take turns and are joined in LDS, a long row is split over workgroups.  One launch holds the rows' own and the
// shared pages.
//
// What bounds it is memory where rows are long, 4 D bytes a token and KV head (32 rows to 8001 tokens, 64 / 8 heads x 128:
// 131 us, 5.1 TB/s of a large copy's 5.0), and otherwise its chain of round trips: queries and lengths, table, first tile,
// join (575 tokens of one row, 32 / 8 x 64: 6 to 6.6 us in a graph, where a launch is 2).
//   * scores are rows = tokens, columns = query heads (v_mfma_f32_16x16x32); a lane then holds 4 + 4 tokens of
//     one column, which is the second operand of the product with V, so weights stay in registers;
//   * K and V come in whole rows and go through the wave's own LDS one after the other, without a barrier: K is read as
//     the first operand, rows 16 bytes further apart than they are long, V back transposed (ds_read_b64_tr_b16: four
//     tokens of a dim to a lane), 32 bytes, so that the rows of a read take all banks alike (operands straight from memory,
//     sixteen bytes of sixteen rows at a time: the batch above 137 us instead of 132);
//   * K of the next tile is requested once LDS holds the present one's, V likewise; the first tile, which every row has,
//     before the row's length is known;
//   * a weight is rounded once to the 16-bit type, half a step, and its sum adds the rounded ones, so that
//     what weights have in common cancels in the quotient; the rest averages out to about what the store's own
//     rounding costs.  (A second part of a weight would be exact to 2^-17, but its product with an infinite value
//     is NaN.)
// Waves: four; eight for lone rows of sixteen columns (see split_few).  Registers: 117 for one block of columns at D = 64 to
// 255 at 256, whose sums lie in the accumulators.
#include "paged_attention.h"

namespace tt {

constexpr int kTile = 32;

__device__ __forceinline__ int over_columns_max(int v) {
#define TT_LEVEL(X) v = max(v, __builtin_bit_cast(int, xor_partner<X>(__builtin_bit_cast(float, v))));
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8)
#undef TT_LEVEL
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ float col_max(float v) {   // over the four lanes of a column
  v = fmaxf(v, xor_partner<16>(v));
  return fmaxf(v, xor_partner<32>(v));
}

// MIXED: a tile's tokens may be seen by some columns and not by others.
template <typename T, int D, int NB, bool MIXED, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : D * NB == 256 || WAVES == 8 ? 2 : 3)))
void paged_few_kernel(PagedParams P) {
  using B = Bits16<T>;
  constexpr int KI = D / 32, VT = D / 16;
  constexpr int PC = D / 8, VR = 64 / PC, VK = 32 / VR;   // pieces of a V row, rows of a request, requests
  constexpr int KS = 2 * D + 16, VS = 2 * D + 32;         // LDS bytes of a row of K, of V
  constexpr int OS = D + 4;                               // floats of a column when the waves are joined
  static_assert(WAVES * 16 * OS * 4 <= WAVES * kTile * VS, "the join fits where V was");
  __shared__ __attribute__((aligned(16))) char lds[WAVES * kTile * VS];
  __shared__ float m_s[WAVES][16], l_s[WAVES][16];
  __shared__ Seen see_s[MIXED ? 16 * NB : 1];
  __shared__ uint32_t marks_s[16 * NB * (D / 16)];
  __shared__ int marked;
  // KV heads and column blocks, rows, splits are the grid's axes; where it holds two jobs, all in x, the shared pages' first
  int x = blockIdx.x, row = blockIdx.y, split = blockIdx.z;
  const bool both = MIXED && P.few[1].blocks > 0, shared_job = both && x < P.few[1].blocks;
  const FewJob J = P.few[shared_job ? 1 : 0];
  if (both) {
    if (!shared_job) x -= P.few[1].blocks;
    const int kvhs = (int)P.c.kv_heads * J.row_tiles, rest = x / kvhs;
    split = rest / J.rows;
    row = rest - split * J.rows;
    x -= rest * kvhs;
  }
  const int kvh = J.row_tiles == 1 ? x : x / J.row_tiles, cb = x - kvh * J.row_tiles;
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = P.per_kv;
  int first = 0, count = P.of.tokens;
  if (!shared_job) {
    first = row * P.of.each;
    count = P.of.each;
    if (MIXED && P.of.cu) count = P.of.count(row, &first);
  }
  const int c0 = cb * 16 * NB, cols = min(16 * NB, count * G - c0);
  if (MIXED && cols <= 0) return;
  const int32_t* table = P.table + (shared_job ? 0 : row * P.table_row);
  const int32_t* sel = P.selected ? P.selected + ((int64_t)row * P.c.kv_heads + kvh) * P.selected_count : nullptr;

  // ---- q, and the first tile where it does not depend on the row's length, are requested before anything else
  int token[NB], head[NB];
  u4_t qb[NB][KI];
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const int c = c0 + min(16 * b + n, cols - 1);
    const int i = MIXED ? c / G : 0;
    token[b] = first + i;
    head[b] = kvh * G + c - i * G;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(P.q) + token[b] * P.q_token + head[b] * P.q_head + 8 * quad;
    if (P.q_vec) {
#pragma unroll
      for (int k = 0; k < KI; k++) qb[b][k] = *reinterpret_cast<const u4_t*>(q + 32 * k);
    } else {
#pragma unroll
      for (int k = 0; k < KI; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) qb[b][k][e] = q[32 * k + 2 * e] | ((uint32_t)q[32 * k + 2 * e + 1] << 16);
    }
  }
  const uint32_t k_step = (uint32_t)(2 * P.c.k_token), v_step = (uint32_t)(2 * P.c.v_token);
  const int v_row = lane / PC, v_piece = lane % PC;
  u4_t kr[VK], vr[VK];
  auto load_k = [&](const Place (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < VK; k++) {
      const int h = k * VR / 16;
      kr[k] = *reinterpret_cast<const u4_t*>(p[h].k + (size_t)((uint32_t)(k * VR - 16 * h + v_row) * k_step + 16 * v_piece));
    }
  };
  auto load_v = [&](const Place (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < VK; k++) {
      const int h = k * VR / 16;
      vr[k] = *reinterpret_cast<const u4_t*>(p[h].v + (size_t)((uint32_t)(k * VR - 16 * h + v_row) * v_step + 16 * v_piece));
    }
  };
  PageLanes lanes{table, P.table, sel, P.shared_entries, P.table_pages, P.selected_count, (int)P.c.pages, 0, {0, 0}, {0, 0}};
  const char* const kbase = reinterpret_cast<const char*>(P.c.k_pages) + 2 * kvh * P.c.k_head;
  const char* const vbase = reinterpret_cast<const char*>(P.c.v_pages) + 2 * kvh * P.c.v_head;
  auto place = [&](int j, Place (&p)[2]) __attribute__((always_inline)) {
    lanes.reach((kTile * j) >> P.page_shift);
    p[0] = place_of(P, lanes, kbase, vbase, kTile * j);
    p[1] = place_of(P, lanes, kbase, vbase, kTile * j + 16);
  };
  // (a place past the table is one in page 0 that nobody sees; a row's first split has a tile unless the row is empty)
  int tile0 = sel || shared_job ? 0 : P.shared / kTile;
  const bool early = split == 0 && (P.window == 0 || sel);
  Place now[2], next[2];
  if (early) {
    lanes.start((kTile * (tile0 + wave)) >> P.page_shift);
    place(tile0 + wave, now);
    load_k(now);
    load_v(now);
    place(tile0 + wave + WAVES, next);
  }

  Seen see[NB];
  int hi_most = 0, hi_least, lo_least, lo_most;             // over the columns
  if (shared_job) {
    int hl = 0x7fffffff, ll = 0x7fffffff, lm = 0;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      int place, each;
      const int r = row_of(P.of, token[b], &place, &each);
      see[b] = r < P.of.rows ? seen_of(P, true, row_length(P, r), place, each) : Seen{0, 0};
      see[b].hi = max(see[b].hi, 0);
      if (see[b].hi > see[b].lo) {         // (one that sees nothing may compute what it will, it ends without weight and maximum)
        hi_most = max(hi_most, see[b].hi); hl = min(hl, see[b].hi);
        ll = min(ll, see[b].lo); lm = max(lm, see[b].lo);
      }
    }
    hi_most = over_columns_max(hi_most);
    lo_most = over_columns_max(lm);
    hi_least = -over_columns_max(-hl);
    lo_least = -over_columns_max(-ll);
  } else {
    const int len = row_length(P, row);
    const int z0 = MIXED ? c0 / G : 0, z1 = MIXED ? (c0 + cols - 1) / G : 0;
#pragma unroll
    for (int b = 0; b < NB; b++) see[b] = seen_of(P, false, len, token[b] - first, count);
    const Seen a = seen_of(P, false, len, z0, count), z = seen_of(P, false, len, z1, count);
    hi_most = max(z.hi, 0); hi_least = a.hi; lo_least = a.lo; lo_most = z.lo;
  }
  int tile1 = (hi_most + kTile - 1) / kTile;
  if (sel) {
    int named = 0;                                           // places of the selection, without those of none at its end
    if (hi_most > 0) {
      for (int e = (P.selected_count - 1) & ~63; e >= 0 && named == 0; e -= 64) {
        const uint64_t any = __builtin_amdgcn_ballot_w64(e + lane < P.selected_count && sel[min(e + lane, P.selected_count - 1)] >= 0);
        if (any != 0) named = e + 64 - __builtin_clzll(any);
      }
    }
    tile1 = ((named << P.page_shift) + kTile - 1) / kTile;
  } else {
    tile0 = lo_least / kTile;
  }
  tile0 += split * J.share;
  tile1 = min(tile1, tile0 + J.share);
  const bool only = P.parts == 1;
  if (tile0 >= tile1) {
    if (!only) {                                             // nothing here: no weight
      for (int c = threadIdx.x; c < cols; c += 64 * WAVES) {
        const int i = (c0 + c) / G;
        P.part_ml[((int64_t)(first + i) * P.heads + kvh * G + (c0 + c - i * G)) * P.parts + J.part0 + split] =
            make_float2(__builtin_bit_cast(float, 0xff800000u), 0.0f);
      }
      return;
    }
    tile1 = tile0;
  }
  int i = tile0 + wave;
  if (!early && tile0 < tile1) {
    lanes.start((kTile * i) >> P.page_shift);
    place(i, now);
    load_k(now);
    load_v(now);
    place(i + WAVES, next);
  }

  // ---- marks
  for (int i = threadIdx.x; i < 16 * NB * (D / 16); i += 64 * WAVES) marks_s[i] = 0;
  if (threadIdx.x == 0) marked = 0;
  if (MIXED && wave == 0 && quad == 0) {
#pragma unroll
    for (int b = 0; b < NB; b++) see_s[16 * b + n] = see[b];
  }
  lds_barrier();
  const Marks marks{marks_s, see_s, cols, D / 16};

  // the sign of the scale goes to q, so that the largest product is the largest score
  const float score_scale = fmaxf(__builtin_fabsf(P.scale_log2), 0x1p-126f);
  if (P.scale_log2 < 0.0f) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int k = 0; k < KI; k++) qb[b][k] ^= 0x80008000u;
  }
  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  f4_t o[NB][VT];
  float m_run[NB], l_run[NB];
#pragma unroll
  for (int b = 0; b < NB; b++) {
#pragma unroll
    for (int x = 0; x < VT; x++) o[b][x] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
    m_run[b] = ninf;
    l_run[b] = 0.0f;
  }
  char* const mine = lds + wave * (kTile * VS);
  char* const k_put = mine + v_row * KS + 16 * v_piece;
  const char* const k_get = mine + n * KS + 16 * quad;
  char* const put = mine + v_row * VS + 16 * v_piece;
  const char* const get = mine + (4 * quad + (n >> 2)) * VS + 8 * (n & 3);

  for (; i < tile1; i += WAVES) {
    f4_t sc[NB][2];
    wave_lds_order();
#pragma unroll
    for (int k = 0; k < VK; k++) *reinterpret_cast<u4_t*>(k_put + k * VR * KS) = kr[k];
    load_k(next);
    wave_lds_order();
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int b = 0; b < NB; b++) sc[b][h] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KI; k++) {
        const u4_t key = *reinterpret_cast<const u4_t*>(k_get + 16 * h * KS + 64 * k);
#pragma unroll
        for (int b = 0; b < NB; b++) sc[b][h] = B::mfma16(key, qb[b][k], sc[b][h]);
      }
    }
    const int t0 = now[0].t, t1 = now[1].t;
    const bool whole = t0 >= lo_most && t0 + 16 <= hi_least && t1 >= lo_most && t1 + 16 <= hi_least;
    if (now[0].bad || now[1].bad) {                          // a column that sees a token in no page is NaN
      if constexpr (MIXED) {
        if (now[0].bad) marks.no_page(t0, 16);
        if (now[1].bad) marks.no_page(t1, 16);
        marked = 1;
      } else if ((now[0].bad && t0 < hi_most && t0 + 16 > lo_least) || (now[1].bad && t1 < hi_most && t1 + 16 > lo_least)) {
        for (int w = lane; w < 16 * NB * (D / 16); w += 64) marks_s[w] = 0xffffffffu;
        marked = 1;
      }
    }
    bool odd = false;
    if (!whole) {
      // tokens out of every column's sight: no value (what lies there may be NaN)
#pragma unroll
      for (int k = 0; k < VK; k++) {
        const int h = k * VR / 16, t = (h ? t1 : t0) + k * VR - 16 * h + v_row;
        if (t < lo_least || t >= hi_most) vr[k] = (u4_t){0u, 0u, 0u, 0u};
        if (MIXED) odd |= any_not_finite<T>(vr[k]);
      }
    }
    wave_lds_order();
#pragma unroll
    for (int k = 0; k < VK; k++) *reinterpret_cast<u4_t*>(put + k * VR * VS) = vr[k];
    if constexpr (MIXED) {
      if (odd) {
        marked = 1;
#pragma unroll 1
        for (int k = 0; k < VK; k++) {
          const int h = k * VR / 16;
          marks.take_odd<T>(reinterpret_cast<uint16_t*>(put + k * VR * VS), (h ? t1 : t0) + k * VR - 16 * h + v_row, 8 * v_piece);
        }
      }
    }
    wave_lds_order();
    load_v(next);
    now[0] = next[0];
    now[1] = next[1];
    if (i + 2 * WAVES < tile1) place(i + 2 * WAVES, next);

    u4_t pw[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      float s[8];
#pragma unroll
      for (int e = 0; e < 8; e++) s[e] = sc[b][e >> 2][e & 3];
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int t = (e < 4 ? t0 : t1) + 4 * quad + (e & 3);
          if (t < see[b].lo || t >= see[b].hi) s[e] = ninf;
        }
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
      // no lane of a column past its maximum by more than the slack: nothing moves
      if (__builtin_amdgcn_ballot_w64(top * score_scale > m_run[b] + kSlack) != 0) {
        const float m_new = fmaxf(m_run[b], col_max(top) * score_scale);
        const float a = m_new == ninf ? 1.0f : __builtin_amdgcn_exp2f(m_run[b] - m_new);
        l_run[b] *= a;
#pragma unroll
        for (int x = 0; x < VT; x++) o[b][x] *= a;
        m_run[b] = m_new;
      }
      const float base = kPScale - (m_run[b] == ninf ? 0.0f : m_run[b]);
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const float pa = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p], score_scale, base));
        const float pb = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p + 1], score_scale, base));
        const uint32_t w = B::pack(pa, pb);
        l_run[b] += lo_f32<T>(w) + hi_f32<T>(w);
        pw[b][p] = w;
      }
    }
#pragma unroll
    for (int x = 0; x < VT; x++) {
      const u2_t va = lds_transposed(get + 32 * x), vb = lds_transposed(get + 16 * VS + 32 * x);
#pragma unroll
      for (int b = 0; b < NB; b++) o[b][x] = B::mfma16((u4_t){va[0], va[1], vb[0], vb[1]}, pw[b], o[b][x]);
    }
  }

  // ---- the waves are joined, sixteen columns at a time
  float* const o_s = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const bool blind = see[b].hi <= see[b].lo;
    const float l_col = blind ? 0.0f : bfly<32>(bfly<16>(l_run[b]));
    __syncthreads();
#pragma unroll
    for (int x = 0; x < VT; x++) *reinterpret_cast<f4_t*>(o_s + (wave * 16 + n) * OS + 16 * x + 4 * quad) = o[b][x];
    if (quad == 0) {
      m_s[wave][n] = blind ? ninf : m_run[b];
      l_s[wave][n] = l_col;
    }
    __syncthreads();
    const int here = min(16, cols - 16 * b);
    for (int u = threadIdx.x; u < here * (D / 4); u += 64 * WAVES) {
      const int cc = u / (D / 4), d = 4 * (u % (D / 4));
      const int c = c0 + 16 * b + cc, at = c / G;
      float M = m_s[0][cc];
#pragma unroll
      for (int w = 1; w < WAVES; w++) M = fmaxf(M, m_s[w][cc]);
      const float base = M == ninf ? 0.0f : M;
      f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) {
        const float e = __builtin_amdgcn_exp2f(m_s[w][cc] - base);
        acc += *reinterpret_cast<const f4_t*>(o_s + (w * 16 + cc) * OS + d) * e;
        l = __builtin_fmaf(l_s[w][cc], e, l);
      }
      const int tok = first + at, hd = kvh * G + c - at * G;
      if (l == 0.0f) acc = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
      if (marked) {
#pragma unroll
        for (int r = 0; r < 4; r++) acc[r] = marks.marked(acc[r], 16 * b + cc, d + r);
      }
      if (only) {
        const float f = finish_scale(P, hd, M, l);
        store_four<T>(reinterpret_cast<T*>(P.out) + tok * P.out_token + hd * P.out_head + d, acc * f, P.out_vec);
      } else {
        const int64_t part = ((int64_t)tok * P.heads + hd) * P.parts + J.part0 + split;
        *reinterpret_cast<f4_t*>(P.part_o + part * D + d) = acc;
        if (d == 0) P.part_ml[part] = make_float2(M, l);
      }
    }
  }
}

template <typename T, int D, int NB>
static int launch_blocks(const PagedParams& P, hipStream_t st, const char* what) {
  const FewJob& own = P.few[0];
  const int kvhs = (int)P.c.kv_heads * own.row_tiles;
  const dim3 grid = P.few[1].blocks > 0 ? dim3((unsigned)(own.blocks + P.few[1].blocks))
                                        : dim3((unsigned)kvhs, (unsigned)own.rows, (unsigned)(own.blocks / kvhs / own.rows));
  const bool mixed = P.few[1].blocks > 0 || P.of.each != 1;
  if constexpr (NB == 1 && D < 256) {
    if (P.wide && !mixed) {
      hipLaunchKernelGGL((paged_few_kernel<T, D, NB, false, 8>), grid, dim3(64 * 8), 0, st, P);
      return check_launch(what);
    }
  }
  if (mixed) hipLaunchKernelGGL((paged_few_kernel<T, D, NB, true, 4>), grid, dim3(64 * 4), 0, st, P);
  else hipLaunchKernelGGL((paged_few_kernel<T, D, NB, false, 4>), grid, dim3(64 * 4), 0, st, P);
  return check_launch(what);
}

template <typename T>
static int launch_type(const PagedParams& P, int blocks16, hipStream_t st, const char* what) {
  if (P.c.head_dim == 64)
    return blocks16 == 1   ? launch_blocks<T, 64, 1>(P, st, what)
           : blocks16 == 2 ? launch_blocks<T, 64, 2>(P, st, what)
                           : launch_blocks<T, 64, 4>(P, st, what);
  if (P.c.head_dim == 128) return blocks16 == 1 ? launch_blocks<T, 128, 1>(P, st, what) : launch_blocks<T, 128, 2>(P, st, what);
  return launch_blocks<T, 256, 1>(P, st, what);
}

int launch_paged_few(const PagedParams& P, int blocks16, hipStream_t st, const char* what) {
  return P.c.dtype == TT_F16 ? launch_type<f16_t>(P, blocks16, st, what) : launch_type<bf16_t>(P, blocks16, st, what);
}

}  // namespace tt
