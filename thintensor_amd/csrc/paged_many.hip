// Paged attention for many columns (chunks of prompts, large batches against their shared pages): a workgroup
// takes 128 or 256 columns of a KV head, 32 for each of its four or eight waves, and walks over the tokens they see,
// 64 at a time (32 with head_dim 256), whose K and V its waves share in LDS.
//
// What bounds it is the matrix cores and, beside them, the vector instructions of the softmax, six for each product
// (4096 queries behind 16384 tokens, 64 / 8 heads: x 128 1967 us, 980 TFLOP/s, x 64 890, x 256 850; a large bf16 product
// reaches 1237); where chunks are short, the start and the end of a workgroup (1024 tokens of one row, 40 / 10 x 128: 43 us).
//   * scores are rows = tokens, columns = query heads (v_mfma_f32_32x32x16), so a column's maximum and sum need
//     one exchange, with lane + 32, and the weights are the second operand of the product with V as they are;
//   * V is read from LDS transposed (ds_read_b64_tr_b16); rows of K lie 16 bytes further apart than they
//     are long, those of V 32, so that the rows of a read take all banks alike;
//   * two buffers, one barrier a tile; the next tile goes to LDS behind the scores' products, the one after it is on its
//     way from memory in registers.  (The waves' halves a phase apart, one with scores while the other weighs, with two
//     barriers a tile: 2262 us against 1967; the matrix cores overlap with other waves' instructions without it.)
//   * values that are not finite are marked where a tile is staged and not in the products, so that no register
//     spills (1159 to 790 us for four chunks to 2048 tokens behind 8192, 40 / 10 x 128);
//   * weights are rounded once to the 16-bit type, and their sum adds the rounded ones (see paged_few.hip).
#include "paged_attention.h"

namespace tt {

// The column tile with the x-th most tokens to see (of up to 64 rows, `count` and `len` of one in each lane; of equal ones the lower row's),
// so that no long one begins when the others end.  Tile j of a row with n of them sees about b + j + 1 times 128 / per_kv
// tokens; how many tiles see h or more is a sum over the rows, and h is found by halving.
template <int COLUMNS>
__device__ __forceinline__ bool longest(const PagedParams& P, int x, int count, int len, int* row, int* tile) {
  const int lane = threadIdx.x & 63;
  int n = count;
  const int64_t before = ((int64_t)max(len - n, 0) * P.per_kv) / COLUMNS;
  const int b = (int)min(before, (int64_t)1 << 29);        // (longer ones need no order, sums of it have to stay in range)
  n = lane < P.of.rows ? (int)(((int64_t)n * P.per_kv + COLUMNS - 1) / COLUMNS) : 0;
  auto at_least = [&](int h) __attribute__((always_inline)) {
    return (int)__builtin_amdgcn_readlane((int)lanes_before((uint32_t)min(max(b + n - h + 1, 0), n)), 63);
  };
  if (x >= at_least(0)) return false;
  int lo = 0, hi = 0x40000000;                 // at_least(lo) > x, at_least(hi) <= x
  {
    int most = n > 0 ? b + n + 1 : 1;
#define TT_LEVEL(X) most = max(most, __builtin_bit_cast(int, xor_partner<X>(__builtin_bit_cast(float, most))));
    TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
    hi = __builtin_amdgcn_readfirstlane(most);
  }
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (at_least(mid) > x) lo = mid;
    else hi = mid;
  }
  uint64_t equal = __builtin_amdgcn_ballot_w64(lo - 1 - b >= 0 && lo - 1 - b < n);
  for (int skip = x - at_least(lo + 1); skip > 0; skip--) equal &= equal - 1;
  if (equal == 0) return false;
  *row = __builtin_ctzll(equal);
  *tile = lo - 1 - __builtin_amdgcn_readlane(b, *row);
  return true;
}

template <typename T, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D == 64 ? (WAVES == 8 ? 4 : 3) : 2)))
void paged_many_kernel(PagedParams P, int splits) {
  using B = Bits16<T>;
  constexpr int COLUMNS = 32 * WAVES;
  constexpr int TT = D == 256 ? 32 : 64, J = TT / 32;
  constexpr int KI = D / 16, VT = D / 32;
  constexpr int PC = D / 8, RR = 64 * WAVES / PC, NK = TT / RR;      // pieces of a row, rows of a request, requests
  constexpr int KS = 2 * D + 16, VS = 2 * D + 32, BUF = TT * (KS + VS);
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF];

  // Workgroups go to the eight XCDs in turn.  Of kvhs = 8 F + R heads an XCD takes F by itself, so that their K and V come
  // to its L2 alone, and an eighth of the tiles of the others; eight tiles of all heads follow the eight before.
  const int kvhs = (int)P.c.kv_heads, xcd = blockIdx.x & 7, i = blockIdx.x >> 3, full = kvhs >> 3;
  int kvh, rest = 8 * (blockIdx.y + gridDim.y * blockIdx.z);
  if (i < 8 * full) {
    const int of = full == 1 ? i : i / full;
    kvh = xcd * full + i - of * full;
    rest += of;
  } else {
    kvh = i;
    rest += (xcd + i) & 7;
  }
  const int x_first = splits == 1 ? rest : rest / splits, split = rest - x_first * splits, x = P.tiles - 1 - x_first;
  if (x < 0) return;
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = P.per_kv;
  int row = 0, first = 0, count = P.of.tokens, len = 0, c0 = x * COLUMNS;
  if (!P.shared_job) {
    if (P.of.rows <= 64 && (P.ordered || P.of.cu)) {       // a row for each lane, what is known of it in one request
      const int r = min(lane, P.of.rows - 1);
      int r_first;
      const int r_count = P.of.count(r, &r_first), r_len = row_length(P, r);
      int tile;
      if (P.ordered) {
        if (!longest<COLUMNS>(P, x_first, r_count, r_len, &row, &tile)) return;
      } else {
        const int before = (int)((int64_t)r_first * G / COLUMNS) + r;
        row = max(0, __popcll(__builtin_amdgcn_ballot_w64(lane < P.of.rows && before <= x)) - 1);
        tile = x - __builtin_amdgcn_readlane(before, row);
      }
      first = __builtin_amdgcn_readlane(r_first, row);
      count = __builtin_amdgcn_readlane(r_count, row);
      len = __builtin_amdgcn_readlane(r_len, row);
      c0 = tile * COLUMNS;
    } else {
      if (P.of.cu) {
        row = P.of.find(x, G, COLUMNS, 1);
        count = P.of.count(row, &first);
        c0 = (x - (int)((int64_t)first * G / COLUMNS) - row) * COLUMNS;
      } else {
        row = x / P.row_tiles;
        count = P.of.each;
        first = row * count;
        c0 = (x - row * P.row_tiles) * COLUMNS;
      }
      len = row_length(P, row);
    }
    row = __builtin_amdgcn_readfirstlane(row);
    first = __builtin_amdgcn_readfirstlane(first);
    count = __builtin_amdgcn_readfirstlane(count);
    len = __builtin_amdgcn_readfirstlane(len);
    c0 = __builtin_amdgcn_readfirstlane(c0);
  }
  const int cols = min(COLUMNS, count * G - c0);
  if (cols <= 0 || c0 < 0) return;

  // ---- columns
  const int c = c0 + min(32 * wave + n, cols - 1), at = c / G;
  const bool mine = 32 * wave + n < cols;
  const int token = first + at, head = kvh * G + c - at * G;
  u4_t qb[KI];
  {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(P.q) + token * P.q_token + head * P.q_head + 8 * half;
    if (P.q_vec) {
#pragma unroll
      for (int k = 0; k < KI; k++) qb[k] = *reinterpret_cast<const u4_t*>(q + 16 * k);
    } else {
#pragma unroll
      for (int k = 0; k < KI; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) qb[k][e] = q[16 * k + 2 * e] | ((uint32_t)q[16 * k + 2 * e + 1] << 16);
    }
  }
  Seen see;
  if (P.shared_job) {
    int place, each;
    const int r = row_of(P.of, token, &place, &each);
    see = r < P.of.rows ? seen_of(P, P.shared_job != 0, row_length(P, r), place, each) : Seen{0, 0};
  } else {
    see = seen_of(P, P.shared_job != 0, len, at, count);
  }
  see.hi = max(see.hi, 0);
  // of this wave's columns, and of all of them
  auto most = [&](int v) __attribute__((always_inline)) {
#define TT_LEVEL(X) v = max(v, __builtin_bit_cast(int, xor_partner<X>(__builtin_bit_cast(float, v))));
    TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16)
#undef TT_LEVEL
    return __builtin_amdgcn_readfirstlane(v);
  };
  // (a column that sees nothing may compute what it will, it ends without weight and maximum)
  constexpr int kFar = 0x7fffffff;
  const bool blind = see.hi <= see.lo;
  const int hi_most = most(blind ? 0 : see.hi), hi_least = -most(blind ? -kFar : -see.hi);
  const int lo_most = most(blind ? 0 : see.lo), lo_least = -most(blind ? -kFar : -see.lo);
  __shared__ int reach[4][WAVES];
  __shared__ Seen see_s[COLUMNS];
  __shared__ uint32_t which_s[COLUMNS];         // a column's token past the first one's, its head in the KV head
  __shared__ uint32_t marks_s[COLUMNS * (D / 16)];
  __shared__ int marked;
  for (int i = threadIdx.x; i < COLUMNS * (D / 16); i += 64 * WAVES) marks_s[i] = 0;
  if (threadIdx.x == 0) marked = 0;
  if (half == 0) {
    see_s[32 * wave + n] = see;
    which_s[32 * wave + n] = ((uint32_t)(at - c0 / G) << 16) | (uint32_t)(c - at * G);
  }
  const Marks marks{marks_s, see_s, cols, D / 16};
  if (lane == 0) {
    reach[0][wave] = -lo_least;
    reach[1][wave] = hi_most;
    reach[2][wave] = lo_most;
    reach[3][wave] = -hi_least;
  }
  __syncthreads();
  auto of_all = [&](int i) __attribute__((always_inline)) {
    int v = reach[i][0];
#pragma unroll
    for (int w = 1; w < WAVES; w++) v = max(v, reach[i][w]);
    return v;
  };
  const int all_lo = -of_all(0), all_hi = of_all(1), part_lo = of_all(2), part_hi = -of_all(3);
  int tile0 = __builtin_amdgcn_readfirstlane(all_lo / TT), tile1 = __builtin_amdgcn_readfirstlane((all_hi + TT - 1) / TT);
  if (splits > 1) {
    // the tiles there are, in even shares
    const int share = max(P.share, (tile1 - tile0 + splits - 1) / splits);
    tile0 += split * share;
    tile1 = min(tile1, tile0 + share);
  }
  const bool only = P.parts == 1;
  const int64_t part = ((int64_t)token * P.heads + head) * P.parts + P.part0 + split;
  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  if (tile0 >= tile1 && !only) {
    if (mine && half == 0) P.part_ml[part] = make_float2(ninf, 0.0f);
    return;
  }

  // A wave brings 64 / PC rows of every request, which lie in one page, so that where they are is the wave's.
  const int32_t* table = P.table + (P.shared_job ? 0 : row * P.table_row);
  const int l_piece = lane % PC, w_row = lane / PC, l_row = wave * (64 / PC) + w_row;
  const uint32_t k_step = (uint32_t)(2 * P.c.k_token), v_step = (uint32_t)(2 * P.c.v_token);
  const uint32_t k_at = (uint32_t)w_row * k_step + 16 * l_piece, v_at = (uint32_t)w_row * v_step + 16 * l_piece;
  const int page_mask = (1 << P.page_shift) - 1;
  const char* const kbase = reinterpret_cast<const char*>(P.c.k_pages) + 2 * kvh * P.c.k_head;
  const char* const vbase = reinterpret_cast<const char*>(P.c.v_pages) + 2 * kvh * P.c.v_head;
  u4_t kr[NK], vr[NK];
  PageLanes lanes{table, P.table, nullptr, P.shared_entries, P.table_pages, 0, (int)P.c.pages, 0, {0, 0}, {0, 0}};
  auto load = [&](int tile) __attribute__((always_inline)) {
    lanes.reach((min(tile, tile1 - 1) * TT) >> P.page_shift);
#pragma unroll
    for (int k = 0; k < NK; k++) {
      const int t = min(tile, tile1 - 1) * TT + k * RR + wave * (64 / PC);
      const int page = lanes.pick(lanes.id, t >> P.page_shift);
      const bool bad = (uint32_t)page >= (uint32_t)P.c.pages;
      if (bad && tile < tile1) {           // (rare, and more than one lane may say so)
        marks.no_page(t, 64 / PC);
        marked = 1;
      }
      const int64_t id = bad ? 0 : page;
      const int64_t slot = t & page_mask;
      kr[k] = *reinterpret_cast<const u4_t*>(kbase + 2 * id * P.c.k_page + slot * k_step + (size_t)k_at);
      vr[k] = *reinterpret_cast<const u4_t*>(vbase + 2 * id * P.c.v_page + slot * v_step + (size_t)v_at);
    }
  };
  // rows outside of every column's sight hold no value; what some columns see and others do not is looked at
  auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
    char* const k_s = lds + buf * BUF + l_row * KS + 16 * l_piece;
    char* const v_s = lds + buf * BUF + TT * KS + l_row * VS + 16 * l_piece;
    const int t0 = tile * TT;
    bool odd = false;
    if (t0 < part_lo || t0 + TT > part_hi) {
#pragma unroll
      for (int k = 0; k < NK; k++) {
        const int t = t0 + k * RR + l_row;
        if (t < all_lo || t >= all_hi) vr[k] = (u4_t){0u, 0u, 0u, 0u};
        odd |= any_not_finite<T>(vr[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NK; k++) {
      *reinterpret_cast<u4_t*>(k_s + k * RR * KS) = kr[k];
      *reinterpret_cast<u4_t*>(v_s + k * RR * VS) = vr[k];
    }
    if (odd) {
      marked = 1;
#pragma unroll 1
      for (int k = 0; k < NK; k++) marks.take_odd<T>(reinterpret_cast<uint16_t*>(v_s + k * RR * VS), t0 + k * RR + l_row, 8 * l_piece);
    }
  };

  const float score_scale = fmaxf(__builtin_fabsf(P.scale_log2), 0x1p-126f);
  if (P.scale_log2 < 0.0f) {
#pragma unroll
    for (int k = 0; k < KI; k++) qb[k] ^= 0x80008000u;
  }
  f16v_t o[VT];
#pragma unroll
  for (int v = 0; v < VT; v++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[v][r] = 0.0f;
  float m_run = ninf, l_run = 0.0f;
  const uint32_t k_get = (uint32_t)(n * KS + 16 * half);
  const uint32_t v_get = (uint32_t)(TT * KS + (4 * half + ((lane & 15) >> 2)) * VS + 32 * ((lane >> 4) & 1) + 8 * (lane & 3));

  if (tile0 < tile1) {
    lanes.start((tile0 * TT) >> P.page_shift);
    load(tile0);
    stage(tile0, 0);
    load(tile0 + 1);
  }
  lds_barrier();
  for (int tile = tile0; tile < tile1; tile++) {
    const int buf = (tile - tile0) & 1, t0 = tile * TT;
    const char* const buf_s = lds + buf * BUF;
    const bool seen = t0 < hi_most && t0 + TT > lo_least;
    f16v_t s[J];
    if (seen) {
#pragma unroll
      for (int j = 0; j < J; j++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[j][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < KI; k++)
          s[j] = B::mfma32(*reinterpret_cast<const u4_t*>(buf_s + k_get + j * 32 * KS + 32 * k), qb[k], s[j]);
      }
    }
    // the next tile goes to LDS while the matrix cores work
    if (tile + 1 < tile1) {
      stage(tile + 1, buf ^ 1);
      load(tile + 2);
    }
    if (seen) {
      if (t0 < lo_most || t0 + TT > hi_least) {
        const int t_lane = t0 + 4 * half - see.lo;
        const uint32_t width = (uint32_t)max(see.hi - see.lo, 0);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            if ((uint32_t)(t_lane + 32 * j + 8 * (r >> 2) + (r & 3)) >= width) s[j][r] = ninf;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int j = 0; j < J; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, s[j][r]);
      if (__builtin_amdgcn_ballot_w64(top * score_scale > m_run + kSlack) != 0) {
        const float m_new = fmaxf(m_run, fmaxf(top, xor_partner<32>(top)) * score_scale);
        const float a = m_new == ninf ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= a;
#pragma unroll
        for (int v = 0; v < VT; v++) o[v] *= a;
        m_run = m_new;
      }
      const float base = kPScale - (m_run == ninf ? 0.0f : m_run);
      float sum = 0.0f;                    // (of a tile: the pair's addition may cut where it should round)
#pragma unroll
      for (int j = 0; j < J; j++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          u4_t p;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][8 * k + 2 * e], score_scale, base));
            const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][8 * k + 2 * e + 1], score_scale, base));
            p[e] = B::pack(a, b);
            sum = B::add_pair(p[e], sum);
          }
          const char* const v_s = buf_s + v_get + (32 * j + 16 * k) * VS;
#pragma unroll
          for (int v = 0; v < VT; v++) {
            const u2_t lo = lds_transposed(v_s + 64 * v), hi = lds_transposed(v_s + 8 * VS + 64 * v);
            o[v] = B::mfma32((u4_t){lo[0], lo[1], hi[0], hi[1]}, p, o[v]);
          }
        }
      l_run += sum;
    }
    lds_barrier();
  }

  // ---- through LDS, so that whole vectors are written: up to 128 dims of the wave's columns at a time
  const float l = blind ? 0.0f : bfly<32>(l_run);
  const float f = only ? finish_scale(P, head, m_run, l) : 1.0f;
  if (!only && mine && half == 0) P.part_ml[part] = make_float2(blind ? ninf : m_run, l);
  const bool any_marks = marked != 0;
  constexpr int DD = WAVES == 8 ? 32 : D, OS = DD + 4, LANES = DD / 4, COLS = 64 / LANES;
  static_assert(WAVES * 32 * OS * 4 <= 2 * BUF, "the wave's sums fit where tiles were");
  float* const o_s = reinterpret_cast<float*>(lds) + wave * 32 * OS;
  const int wave_cols = min(32, cols - 32 * wave), y_col = lane / LANES, y_dim = 4 * (lane % LANES);
#pragma unroll
  for (int v0 = 0; v0 < VT; v0 += DD / 32) {
    wave_lds_order();
#pragma unroll
    for (int v = 0; v < DD / 32; v++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        f4_t y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = l == 0.0f ? 0.0f : o[v0 + v][4 * r + e] * f;
        *reinterpret_cast<f4_t*>(o_s + n * OS + 32 * v + 8 * r + 4 * half) = y;
      }
    wave_lds_order();
#pragma unroll 4
    for (int i = y_col; i < wave_cols; i += COLS) {
      f4_t y = *reinterpret_cast<const f4_t*>(o_s + i * OS + y_dim);
      const int d = 32 * v0 + y_dim;
      if (any_marks) {
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = marks.marked(y[e], 32 * wave + i, d + e);
      }
      const uint32_t which = which_s[32 * wave + i];
      const int tok = first + c0 / G + (int)(which >> 16), hd = kvh * G + (int)(which & 0xffffu);
      if (only) store_four<T>(reinterpret_cast<T*>(P.out) + tok * P.out_token + hd * P.out_head + d, y, P.out_vec);
      else *reinterpret_cast<f4_t*>(P.part_o + (((int64_t)tok * P.heads + hd) * P.parts + P.part0 + split) * D + d) = y;
    }
  }
}

template <typename T, int D>
static int launch_dim(const PagedParams& P, int waves, int splits, hipStream_t st, const char* what) {
  const unsigned eights = ((unsigned)P.tiles * splits + 7) / 8, most = 32768;
  const dim3 grid((unsigned)P.c.kv_heads * 8, eights < most ? eights : most, (eights + most - 1) / most);
  if constexpr (D < 256) {
    if (waves == 4) {
      hipLaunchKernelGGL((paged_many_kernel<T, D, 4>), grid, dim3(64 * 4), 0, st, P, splits);
      return check_launch(what);
    }
  }
  hipLaunchKernelGGL((paged_many_kernel<T, D, 8>), grid, dim3(64 * 8), 0, st, P, splits);
  return check_launch(what);
}

template <typename T>
static int launch_type(const PagedParams& P, int waves, int splits, hipStream_t st, const char* what) {
  if (P.c.head_dim == 64) return launch_dim<T, 64>(P, waves, splits, st, what);
  if (P.c.head_dim == 128) return launch_dim<T, 128>(P, waves, splits, st, what);
  return launch_dim<T, 256>(P, waves, splits, st, what);
}

int launch_paged_many(const PagedParams& P, int waves, int splits, hipStream_t st, const char* what) {
  return P.c.dtype == TT_F16 ? launch_type<f16_t>(P, waves, splits, st, what) : launch_type<bf16_t>(P, waves, splits, st, what);
}

}  // namespace tt
