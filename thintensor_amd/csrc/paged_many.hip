// Paged attention for many columns (chunks of prompts, large batches against their shared pages): a
// workgroup takes 128 columns of a KV head, 32 for each wave, and walks over the tokens they see, 64 at a
// time (32 with head_dim 256), whose K and V its waves share in LDS.
//
// What bounds it is the matrix cores and, beside them, the vector instructions of the softmax:
//   * scores are rows = tokens, columns = query heads (v_mfma_f32_32x32x16), so a column's maximum and sum need
//     one exchange, with lane + 32, and the weights are the second operand of the product with V as they are;
//   * V is read from LDS transposed (ds_read_b64_tr_b16); rows of K lie 16 bytes further apart than they
//     are long, those of V 32, so that the rows of a read take all banks alike;
//   * two buffers, one barrier a tile; the tile after next is on its way from memory in registers;
//   * weights are rounded once to the 16-bit type, and their sum adds the rounded ones (see paged_few.hip).
#include "paged_attention.h"

namespace tt {

constexpr int kWaves = 4;

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void paged_many_kernel(PagedParams P, int splits) {
  using B = Bits16<T>;
  constexpr int TT = D == 256 ? 32 : 64, J = TT / 32;
  constexpr int KI = D / 16, VT = D / 32;
  constexpr int PC = D / 8, RR = 64 * kWaves / PC, NK = TT / RR;      // pieces of a row, rows of a request, requests
  constexpr int KS = 2 * D + 16, VS = 2 * D + 32, BUF = TT * (KS + VS);
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF];

  const int kvhs = (int)P.c.kv_heads, kvh = blockIdx.x % kvhs;
  const int rest = blockIdx.x / kvhs, split = rest % splits, x = P.tiles - 1 - rest / splits;   // long rows' ends first
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int G = P.per_kv;
  int row = 0, first = 0, count = P.of.tokens, c0 = x * kManyColumns;
  if (!P.shared_job) {
    if (P.of.cu) {
      row = P.of.find(x, G, kManyColumns, 1);
      count = P.of.count(row, &first);
      c0 = (x - (int)((int64_t)first * G / kManyColumns) - row) * kManyColumns;
    } else {
      row = x / P.row_tiles;
      count = P.of.each;
      first = row * count;
      c0 = (x - row * P.row_tiles) * kManyColumns;
    }
    row = __builtin_amdgcn_readfirstlane(row);
    first = __builtin_amdgcn_readfirstlane(first);
    count = __builtin_amdgcn_readfirstlane(count);
    c0 = __builtin_amdgcn_readfirstlane(c0);
  }
  const int cols = min(kManyColumns, count * G - c0);
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
    see = r < P.of.rows ? seen_of(P, row_length(P, r), place, each) : Seen{0, 0};
  } else {
    see = seen_of(P, row_length(P, row), at, count);
  }
  see.hi = max(see.hi, 0);
  // of this wave's columns, and of all of them
  auto most = [&](int v) __attribute__((always_inline)) {
#define TT_LEVEL(X) v = max(v, __builtin_bit_cast(int, xor_partner<X>(__builtin_bit_cast(float, v))));
    TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16)
#undef TT_LEVEL
    return __builtin_amdgcn_readfirstlane(v);
  };
  const int hi_most = most(see.hi), hi_least = -most(-see.hi), lo_most = most(see.lo), lo_least = -most(-see.lo);
  __shared__ int reach[4][kWaves];
  __shared__ Seen see_s[kManyColumns];
  __shared__ uint32_t marks_s[kManyColumns * (D / 16)];
  __shared__ int marked;
  for (int i = threadIdx.x; i < kManyColumns * (D / 16); i += 64 * kWaves) marks_s[i] = 0;
  if (threadIdx.x == 0) marked = 0;
  if (half == 0) see_s[32 * wave + n] = see;
  const Marks marks{marks_s, see_s, cols, D / 16};
  if (lane == 0) {
    reach[0][wave] = -lo_least;
    reach[1][wave] = hi_most;
    reach[2][wave] = lo_most;
    reach[3][wave] = -hi_least;
  }
  __syncthreads();
  auto of_all = [&](int i) __attribute__((always_inline)) { return max(max(reach[i][0], reach[i][1]), max(reach[i][2], reach[i][3])); };
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
  int ids[NK];
  auto look = [&](int tile) __attribute__((always_inline)) {      // the pages of a tile's rows
#pragma unroll
    for (int k = 0; k < NK; k++) {
      const int t = min(tile, tile1 - 1) * TT + k * RR + wave * (64 / PC);
      ids[k] = table[min(t >> P.page_shift, P.table_pages - 1)];
    }
  };
  auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < NK; k++) {
      const int t = min(tile, tile1 - 1) * TT + k * RR + wave * (64 / PC);
      const bool bad = (uint32_t)ids[k] >= (uint32_t)P.c.pages;
      if (bad && tile < tile1) {           // (rare, and more than one lane may say so)
        marks.no_page(t, 64 / PC);
        marked = 1;
      }
      const int64_t id = bad ? 0 : ids[k];
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
    look(tile0);
    load(tile0);
    look(tile0 + 1);
    stage(tile0, 0);
    load(tile0 + 1);
    look(tile0 + 2);
  }
  lds_barrier();
  for (int tile = tile0; tile < tile1; tile++) {
    const int buf = (tile - tile0) & 1, t0 = tile * TT;
    if (tile + 1 < tile1) {
      stage(tile + 1, buf ^ 1);
      load(tile + 2);
      look(tile + 3);
    }
    const char* const buf_s = lds + buf * BUF;
    if (t0 < hi_most && t0 + TT > lo_least) {
      f16v_t s[J];
#pragma unroll
      for (int j = 0; j < J; j++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[j][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < KI; k++)
          s[j] = B::mfma32(*reinterpret_cast<const u4_t*>(buf_s + k_get + j * 32 * KS + 32 * k), qb[k], s[j]);
      }
      if (t0 < lo_most || t0 + TT > hi_least) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int t = t0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
            if (t < see.lo || t >= see.hi) s[j][r] = ninf;
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

  const float l = bfly<32>(l_run);
  if (!mine) return;
  const bool any_marks = marked != 0;
  const float f = only ? finish_scale(P, head, m_run, l) : 1.0f;
  T* out = reinterpret_cast<T*>(P.out) + token * P.out_token + head * P.out_head;
  float* po = P.part_o + part * D;
  if (!only && half == 0) P.part_ml[part] = make_float2(m_run, l);
#pragma unroll
  for (int v = 0; v < VT; v++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int d = 32 * v + 8 * r + 4 * half;
      f4_t y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        y[e] = l == 0.0f ? 0.0f : o[v][4 * r + e] * f;
        if (any_marks) y[e] = marks.marked(y[e], 32 * wave + n, d + e);
      }
      if (only) store_four<T>(out + d, y, P.out_vec);
      else *reinterpret_cast<f4_t*>(po + d) = y;
    }
}

template <typename T>
static int launch_type(const PagedParams& P, int splits, hipStream_t st, const char* what) {
  const dim3 grid((unsigned)(P.c.kv_heads * P.tiles * splits)), block(64 * kWaves);
  if (P.c.head_dim == 64) hipLaunchKernelGGL((paged_many_kernel<T, 64>), grid, block, 0, st, P, splits);
  else if (P.c.head_dim == 128) hipLaunchKernelGGL((paged_many_kernel<T, 128>), grid, block, 0, st, P, splits);
  else hipLaunchKernelGGL((paged_many_kernel<T, 256>), grid, block, 0, st, P, splits);
  return check_launch(what);
}

int launch_paged_many(const PagedParams& P, int splits, hipStream_t st, const char* what) {
  return P.c.dtype == TT_F16 ? launch_type<f16_t>(P, splits, st, what) : launch_type<bf16_t>(P, splits, st, what);
}

}  // namespace tt
