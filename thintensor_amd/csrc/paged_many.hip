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

  const int32_t* table = P.table + (P.shared_job ? 0 : row * P.table_row);
  const int l_row = threadIdx.x / PC, l_piece = threadIdx.x % PC;
  const int page_mask = (1 << P.page_shift) - 1;
  const uint32_t k_step = (uint32_t)(2 * P.c.k_token), v_step = (uint32_t)(2 * P.c.v_token);
  const char* const kbase = reinterpret_cast<const char*>(P.c.k_pages) + 2 * kvh * P.c.k_head + 16 * l_piece;
  const char* const vbase = reinterpret_cast<const char*>(P.c.v_pages) + 2 * kvh * P.c.v_head + 16 * l_piece;
  u4_t kr[NK], vr[NK];
  int ids[NK];
  auto look = [&](int tile) __attribute__((always_inline)) {      // the pages of a tile's rows
#pragma unroll
    for (int k = 0; k < NK; k++) {
      const int t = min(tile, tile1 - 1) * TT + k * RR + l_row;
      ids[k] = table[min(max(t >> P.page_shift, 0), P.table_pages - 1)];
    }
  };
  uint64_t bad_now = 0;                    // whether a row of the loaded tile is in no page
  auto load = [&](int tile) __attribute__((always_inline)) {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < NK; k++) {
      const uint32_t slot = (uint32_t)((min(tile, tile1 - 1) * TT + k * RR + l_row) & page_mask);
      const bool b = (uint32_t)ids[k] >= (uint32_t)P.c.pages;
      const int64_t id = b ? 0 : ids[k];
      bad |= b;
      kr[k] = *reinterpret_cast<const u4_t*>(kbase + 2 * id * P.c.k_page + (size_t)(slot * k_step));
      vr[k] = *reinterpret_cast<const u4_t*>(vbase + 2 * id * P.c.v_page + (size_t)(slot * v_step));
    }
    return bad;
  };
  // Of a buffer: a row in no page, a value that is not finite.  Once set they stay: later tiles then are
  // looked at more closely than they need.
  __shared__ int flags[2][2];
  if (threadIdx.x < 4) flags[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  __syncthreads();
  // rows outside of every column's sight hold no value; what a partly seen tile holds is looked at
  auto stage = [&](int tile, int buf, bool bad) __attribute__((always_inline)) {
    char* const k_s = lds + buf * BUF + l_row * KS + 16 * l_piece;
    char* const v_s = lds + buf * BUF + TT * KS + l_row * VS + 16 * l_piece;
    const int t0 = tile * TT;
    if (t0 < part_lo || t0 + TT > part_hi) {
      bool odd = false;
#pragma unroll
      for (int k = 0; k < NK; k++) {
        const int t = t0 + k * RR + l_row;
        if (t < all_lo || t >= all_hi) vr[k] = (u4_t){0u, 0u, 0u, 0u};
        odd |= any_not_finite<T>(vr[k]);
      }
      if (odd) flags[buf][1] = 1;
    }
#pragma unroll
    for (int k = 0; k < NK; k++) {
      *reinterpret_cast<u4_t*>(k_s + k * RR * KS) = kr[k];
      *reinterpret_cast<u4_t*>(v_s + k * RR * VS) = vr[k];
    }
    if (bad) flags[buf][0] = 1;
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

  bool bad_next = false;
  if (tile0 < tile1) {
    look(tile0);
    bool bad = load(tile0);
    look(tile0 + 1);
    stage(tile0, 0, bad);
    bad_next = load(tile0 + 1);
    look(tile0 + 2);
  }
  lds_barrier();
  for (int tile = tile0; tile < tile1; tile++) {
    const int buf = (tile - tile0) & 1, t0 = tile * TT;
    const bool bad = flags[buf][0] != 0, odd_tile = flags[buf][1] != 0;
    if (tile + 1 < tile1) {
      stage(tile + 1, buf ^ 1, bad_next);
      bad_next = load(tile + 2);
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
      const bool whole = t0 >= lo_most && t0 + TT <= hi_least && !bad;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int t = t0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
            if (bad && (uint32_t)table[min(t >> P.page_shift, P.table_pages - 1)] >= (uint32_t)P.c.pages)
              s[j][r] = __builtin_bit_cast(float, 0x7fc00000u);
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
      const bool odd = odd_tile && !whole;
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
            l_run += lo_f32<T>(p[e]) + hi_f32<T>(p[e]);
          }
          const char* const v_s = buf_s + v_get + (32 * j + 16 * k) * VS;
          if (!odd) {
#pragma unroll
            for (int v = 0; v < VT; v++) {
              const u2_t lo = lds_transposed(v_s + 64 * v), hi = lds_transposed(v_s + 8 * VS + 64 * v);
              o[v] = B::mfma32((u4_t){lo[0], lo[1], hi[0], hi[1]}, p, o[v]);
            }
          } else {
            u4_t vis;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              vis[e] = 0;
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const int r = 8 * k + 2 * e + h, t = t0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
                if (t >= see.lo && t < see.hi) vis[e] |= (uint32_t)B::kOne << (16 * h);
              }
            }
#pragma unroll
            for (int v = 0; v < VT; v++) {
              const u2_t lo = lds_transposed(v_s + 64 * v), hi = lds_transposed(v_s + 8 * VS + 64 * v);
              __builtin_amdgcn_sched_barrier(0);     // one at a time: rare, and should cost no registers
              u4_t clean, code;
              take_odd<T>((u4_t){lo[0], lo[1], hi[0], hi[1]}, clean, code);
              o[v] = B::mfma32(clean, p, o[v]);
              f16v_t count;
#pragma unroll
              for (int r = 0; r < 16; r++) count[r] = 0.0f;
              count = B::mfma32(code, vis, count);
#pragma unroll
              for (int r = 0; r < 16; r++) o[v][r] = with_odd(o[v][r], count[r]);
            }
          }
        }
    }
    lds_barrier();
  }

  const float l = bfly<32>(l_run);
  if (!mine) return;
  if (only) {
    const float f = finish_scale(P, head, m_run, l);
    T* out = reinterpret_cast<T*>(P.out) + token * P.out_token + head * P.out_head;
#pragma unroll
    for (int v = 0; v < VT; v++)
#pragma unroll
      for (int r = 0; r < 16; r++) store<T>(out + 32 * v + 8 * (r >> 2) + 4 * half + (r & 3), l == 0.0f ? 0.0f : o[v][r] * f);
  } else {
    float* po = P.part_o + part * D;
#pragma unroll
    for (int v = 0; v < VT; v++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        *reinterpret_cast<f4_t*>(po + 32 * v + 8 * r + 4 * half) = (f4_t){o[v][4 * r], o[v][4 * r + 1], o[v][4 * r + 2], o[v][4 * r + 3]};
    if (half == 0) P.part_ml[part] = make_float2(m_run, l);
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
