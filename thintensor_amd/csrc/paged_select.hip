// Selecting the pages that a query reads by the bounds of their keys.
#include "paged_attention.h"

namespace tt {

struct SelectParams {
  tt_paged_cache c;
  const void* q;
  int64_t q_token, q_head;
  const int32_t* table;
  int64_t table_row;
  int table_pages, page_shift;
  const int32_t* lengths;
  int max_length, per_kv, first, last, count;
  uint32_t* keys;              // scores as integers in their order
  int64_t keys_row;            // of one (row, KV head)
  int32_t* selected;
};

__device__ __forceinline__ int row_pages(const SelectParams& P, int row) {
  const int n = min(max(P.lengths[row], 0), P.max_length);
  return (n + (1 << P.page_shift) - 1) >> P.page_shift;
}

// Scores as integers in their order; +0 and -0 are equal, NaN comes last.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Scores.  A workgroup takes 64 pages of a row and KV head, whose bounds it brings to LDS in whole rows; a lane then
// has a page and a wave a quarter of the dims.  max(q low, q high) = q (high + low) / 2 + |q| (high - low) / 2, two
// binary64 fmas with what LDS holds of half the queries, the same for all lanes; both are exact but for the addition.
// With bounds or queries that are not finite the equation fails, and such lanes form their sums once more by the
// definition.  What bounds it is memory where there are many pages, 4 D bytes each, and the reads of the queries.  (8 x 10 x 2048 pages of 128, four
// heads each: lanes that read their own pages' bounds in turns of sixteen bytes, 43 us, since every line came to the CU
// four times over; queries through scalar registers, 103; two pages a lane, with room for one workgroup in LDS, 47; now
// 26, its bytes 17.)
template <typename T, int D, int GH>
__global__ __launch_bounds__(256) void page_score_kernel(SelectParams P) {
  constexpr int QD = D / 4, PIECES = QD / 8;
  constexpr int RP = D / 4, RR = 256 / RP, NR = 64 / RR;      // pieces of a page's bounds, pages of a request, requests
  constexpr int BS = 4 * D + 16;                                   // LDS bytes of a page: reads of a column take all banks alike
  typedef double d2_t __attribute__((ext_vector_type(2)));
  __shared__ __attribute__((aligned(16))) char b_s[64 * BS];
  __shared__ __attribute__((aligned(16))) double q_s[D][GH];       // halves
  __shared__ double part_s[4][GH][64];
  __shared__ int odd_q;
  const int row = blockIdx.z, kvh = blockIdx.y, p0 = blockIdx.x * 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int pages = row_pages(P, row);
  // (entries past the row's pages may be anything, what they lead to is not used)
  auto page_of = [&](int p) __attribute__((always_inline)) {
    const int32_t id = P.table[row * P.table_row + min(p, P.table_pages - 1)];
    return id < 0 || id >= P.c.pages ? -1 : id;
  };
  if (p0 > 0 && p0 >= pages) return;       // the first ones do not wait for the length
  // the queries of a turn: heads past the last repeat it, which changes no maximum
  constexpr int MINE = (GH * D + 255) / 256;
  T qv[MINE];
  auto load_q = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      const int u = threadIdx.x + 256 * i;
      const int h = min(h0 + u / D, P.per_kv - 1), d = u % D;
      qv[i] = reinterpret_cast<const T*>(P.q)[row * P.q_token + (kvh * P.per_kv + h) * P.q_head + d];
    }
  };
  load_q(0);
  {
    const int l_row = threadIdx.x / RP, l_piece = threadIdx.x % RP;
    const char* base = reinterpret_cast<const char*>(P.c.k_bounds) + 2 * kvh * P.c.b_head + 16 * l_piece;
    constexpr int AT_ONCE = NR < 8 ? NR : 8;
#pragma unroll
    for (int r0 = 0; r0 < NR; r0 += AT_ONCE) {
      u4_t v[AT_ONCE];
#pragma unroll
      for (int r = 0; r < AT_ONCE; r++)
        v[r] = *reinterpret_cast<const u4_t*>(base + 2 * (int64_t)max(page_of(p0 + (r0 + r) * RR + l_row), 0) * P.c.b_page);
#pragma unroll
      for (int r = 0; r < AT_ONCE; r++) *reinterpret_cast<u4_t*>(b_s + ((r0 + r) * RR + l_row) * BS + 16 * l_piece) = v[r];
    }
  }
  if (pages <= P.count) return;            // every page is kept, whatever its score
  const char* const mine = b_s + lane * BS + 2 * wave * QD;
  uint32_t best = 0;
  for (int h0 = 0; h0 < P.per_kv; h0 += GH) {
    __syncthreads();
    if (threadIdx.x == 0) odd_q = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      const int u = threadIdx.x + 256 * i;
      const float x = to_f32(qv[i]);
      if (!(__builtin_fabsf(x) < __builtin_bit_cast(float, 0x7f800000u))) odd_q = 1;
      q_s[u % D][u / D] = 0.5 * (double)x;
    }
    if (h0 + GH < P.per_kv) load_q(h0 + GH);
    __syncthreads();
    double sum[GH];
#pragma unroll
    for (int h = 0; h < GH; h++) sum[h] = 0.0;
    bool odd = false;
#pragma unroll 1
    for (int x = 0; x < PIECES; x++) {
      const u4_t lo = *reinterpret_cast<const u4_t*>(mine + 16 * x), hi = *reinterpret_cast<const u4_t*>(mine + 2 * D + 16 * x);
      odd |= any_not_finite<T>(lo) || any_not_finite<T>(hi);
      const double* q = q_s[wave * QD + 8 * x];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double a = (double)((e & 1) ? hi_f32<T>(lo[e >> 1]) : lo_f32<T>(lo[e >> 1]));
        const double b = (double)((e & 1) ? hi_f32<T>(hi[e >> 1]) : lo_f32<T>(hi[e >> 1]));
#pragma unroll
        for (int h = 0; h < GH; h += 2) {
          const d2_t qq = *reinterpret_cast<const d2_t*>(q + GH * e + h);
#pragma unroll
          for (int i = 0; i < 2; i++)
            sum[h + i] = __builtin_fma(__builtin_fabs(qq[i]), b - a, __builtin_fma(qq[i], b + a, sum[h + i]));
        }
      }
    }
#pragma unroll
    for (int h = 0; h < GH; h++) part_s[wave][h][lane] = sum[h];
    if (odd || odd_q != 0) {
      const T* at = reinterpret_cast<const T*>(mine);
#pragma unroll 1
      for (int h = 0; h < GH; h++) {
        double t = 0.0;
#pragma unroll 1
        for (int d = 0; d < QD; d++) {
          const double q = 2.0 * q_s[wave * QD + d][h], x = q * (double)to_f32(at[d]), y = q * (double)to_f32(at[D + d]);
          t += x > y || x != x ? x : y;
        }
        part_s[wave][h][lane] = t;
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
#pragma unroll
      for (int h = 0; h < GH; h++) {
        const int at = threadIdx.x;
        const uint32_t k = score_key((float)((part_s[0][h][at] + part_s[1][h][at]) + (part_s[2][h][at] + part_s[3][h][at])));
        best = k > best ? k : best;
      }
    }
  }
  const int p = p0 + threadIdx.x;
  if (threadIdx.x < 64 && p < pages)
    P.keys[((int64_t)row * P.c.kv_heads + kvh) * P.keys_row + p] = page_of(p) < 0 ? 0xffffffffu : best;
}

// The least kept score is found digit by digit: digits of eight bits of key - least key, from the highest that is set
// anywhere, so that the first one already spreads; histograms in LDS, one for each digit, searched by every wave for
// itself, so that a digit takes one barrier.  Then every thread counts what is kept of its run of pages, and the runs
// are written one after another.  Keys stay in registers up to HELD a thread.  What bounds it is the chain of
// barriers and round trips.
template <int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void page_pick_kernel(SelectParams P) {
  constexpr int WAVES = THREADS / 64;
  __shared__ __attribute__((aligned(16))) uint32_t hist[4][256];
  __shared__ uint32_t ends[2][WAVES], counts[2][WAVES];
  const int row = blockIdx.y, kvh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t at = (int64_t)row * P.c.kv_heads + kvh;
  const uint32_t* keys = P.keys + at * P.keys_row;
  int32_t* out = P.selected + at * P.count;
  const int pages = row_pages(P, row), first = min(P.first, pages), last = max(first, pages - P.last);
  const int places = P.count - (first + pages - last);
  // runs of pages by the most there may be, so that keys are requested before the row's length is known (what lies past
  // its pages is not used)
  const int per = ((int)P.keys_row + THREADS - 1) / THREADS, p0 = tid * per, p1 = min(p0 + per, pages);
  uint32_t held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; k++) held[k] = keys[min(p0 + k, (int)P.keys_row - 1)];
  for (int i = tid; i < 4 * 256; i += THREADS) (&hist[0][0])[i] = 0;
  auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < HELD; k++)
      if (p0 + k < p1) f(p0 + k, held[k]);
    for (int p = p0 + HELD; p < p1; p++) f(p, keys[p]);
  };
  // kept: the forced ones, keys past `least`, and the first `want` of those that equal it
  uint32_t least = 0;
  int want = 0;
  if (places >= last - first) {
    want = last - first;                     // everything: equal ones are all that are not greater
    least = 0xffffffffu;
  } else if (places > 0) {
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](int p, uint32_t k) {
      if (p >= first && p < last) {
        lo = min(lo, k);
        hi = max(hi, k);
      }
    });
    lo = ~(uint32_t)(wave_max_u64(~lo));
    hi = (uint32_t)wave_max_u64(hi);
    if (lane == 0) {
      ends[0][wave] = lo;
      ends[1][wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
      lo = min(lo, ends[0][w]);
      hi = max(hi, ends[1][w]);
    }
    uint32_t prefix = 0, mask = 0;
    int shift = hi > lo ? max(0, 24 - __builtin_clz(hi - lo)) : 0;
    want = places;
#pragma unroll 1
    for (int step = 0; step < 4; step++) {
      uint32_t* const h = hist[step];
      each([&](int p, uint32_t k) {
        const uint32_t x = k - lo;
        if (p >= first && p < last && (x & mask) == prefix) atomicAdd(&h[(x >> shift) & 255], 1u);
      });
      __syncthreads();
      // lane l holds the four bins from 252 - 4 l on, so that sums over the lanes run from the top
      const u4_t bins = *reinterpret_cast<const u4_t*>(h + 252 - 4 * lane);
      const uint32_t four = bins[0] + bins[1] + bins[2] + bins[3];
      const uint32_t upto = lanes_before(four), above = upto - four;
      const uint64_t reached = __builtin_amdgcn_ballot_w64(upto >= (uint32_t)want);
      const int where = __builtin_ctzll(reached);
      uint32_t digit = 0, over = above;
      bool done = false;
#pragma unroll
      for (int i = 3; i >= 0; i--) {
        if (!done && over + bins[i] >= (uint32_t)want) {
          digit = 252 - 4 * lane + i;
          done = true;
        }
        if (!done) over += bins[i];
      }
      digit = __builtin_amdgcn_readlane(digit, where);
      over = __builtin_amdgcn_readlane(over, where);
      prefix |= digit << shift;
      mask |= 255u << shift;
      want -= (int)over;
      if (shift == 0) break;
      // the next eight bits; the last digit may repeat some of those before
      shift = max(0, shift - 8);
    }
    least = prefix + lo;
  } else {
    least = 0xffffffffu;
  }
  auto kind = [&](int p, uint32_t k) __attribute__((always_inline)) {      // 2: kept, 1: if among the first
    if (p < first || p >= last) return 2;
    if (places >= last - first) return 2;
    return places <= 0 ? 0 : k > least ? 2 : k == least ? 1 : 0;
  };
  uint32_t greater = 0, equal = 0;
  each([&](int p, uint32_t k) {
    const int c = kind(p, k);
    greater += c == 2;
    equal += c == 1;
  });
  const uint32_t g = lanes_before(greater), e = lanes_before(equal);
  if (lane == 63) {
    counts[0][wave] = g;
    counts[1][wave] = e;
  }
  __syncthreads();
  uint32_t put = g - greater, eq = e - equal, kept = 0, ties = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    const uint32_t a = counts[0][w], b = counts[1][w];
    if (w < wave) {
      put += a;
      eq += b;
    }
    kept += a;
    ties += b;
  }
  put += min(eq, (uint32_t)want);
  each([&](int p, uint32_t k) {
    const int c = kind(p, k);
    const bool keep = c == 2 || (c == 1 && eq < (uint32_t)want);
    eq += c == 1;
    if (keep) out[put++] = p;
  });
  for (int i = (int)(kept + min(ties, (uint32_t)want)) + tid; i < P.count; i += THREADS) out[i] = -1;
}

template <typename T, int D, int GH>
static void launch_score(const SelectParams& P, int64_t most, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)((most + 63) / 64), (unsigned)P.c.kv_heads, (unsigned)rows);
  hipLaunchKernelGGL((page_score_kernel<T, D, GH>), grid, dim3(256), 0, st, P);
}
template <typename T, int D>
static void launch_score(const SelectParams& P, int64_t most, int64_t rows, hipStream_t st) {
  if (P.per_kv <= 4) launch_score<T, D, 4>(P, most, rows, st);
  else launch_score<T, D, 8>(P, most, rows, st);
}
template <typename T>
static void launch_score(const SelectParams& P, int64_t most, int64_t rows, hipStream_t st) {
  if (P.c.head_dim == 64) launch_score<T, 64>(P, most, rows, st);
  else if (P.c.head_dim == 128) launch_score<T, 128>(P, most, rows, st);
  else launch_score<T, 256>(P, most, rows, st);
}

static int check_select(const tt_paged_cache* c, int64_t table_pages, int64_t rows, int64_t heads, int64_t max_length,
                        const char* what) {
  const int rc = check_rows(c, table_pages, false, rows, rows, heads, what);
  if (rc) return rc;
  TT_REQUIRE(c->k_bounds, "%s: the cache keeps no k_bounds", what);
  TT_REQUIRE(max_length >= (rows > 0), "%s: max_length must be at least 1", what);
  return TT_OK;
}

static int64_t most_pages(const tt_paged_cache* c, int64_t table_pages, int64_t max_length) {
  const int64_t p = (max_length - 1) / c->page_size + 1;
  return p < table_pages ? p : table_pages;
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_select_pages_scratch_floats(const tt_paged_cache* cache, int64_t table_pages, int64_t rows, int64_t max_length) {
  if (check_select(cache, table_pages, rows, 0, max_length, "select_pages") != TT_OK) return TT_ERR_INVALID;
  return rows * cache->kv_heads * most_pages(cache, table_pages, max_length);
}

extern "C" int tt_select_pages(const tt_paged_cache* cache, const void* q, int64_t q_token, int64_t q_head,
                               const int32_t* table, int64_t table_row, int64_t table_pages, const int32_t* lengths,
                               int64_t rows, int64_t heads, int64_t first_pages, int64_t last_pages, int64_t max_length,
                               float* scratch, int64_t scratch_floats, int32_t* selected, int64_t selected_count,
                               void* stream) {
  const char* what = "select_pages";
  const int rc = check_select(cache, table_pages, rows, heads, max_length, what);
  if (rc) return rc;
  TT_REQUIRE(heads > 0, "%s: heads must be a multiple of kv_heads", what);
  TT_REQUIRE(first_pages >= 0 && last_pages >= 0 && selected_count >= 1 && selected_count <= 4096 &&
                 first_pages <= selected_count && last_pages <= selected_count - first_pages,
             "%s: count must be at least first_pages + last_pages and 1 to 4096", what);
  if (rows == 0) return TT_OK;
  TT_REQUIRE(q && table && lengths && selected && scratch, "%s: null pointer", what);
  const int64_t most = most_pages(cache, table_pages, max_length);
  TT_REQUIRE(scratch_floats >= rows * cache->kv_heads * most, "%s: scratch too small", what);
  const Region made(selected, 4, selected_count, {{rows, cache->kv_heads * selected_count}, {cache->kv_heads, selected_count}});
  TT_REQUIRE(PagedRegions(cache).apart_from(made) && apart(made, {q, 2, cache->head_dim, {{rows, q_token}, {heads, q_head}}}) &&
                 apart(made, {table, 4, table_pages, {{rows, table_row}}}) && apart(made, {lengths, 4, rows, {}}) &&
                 apart(made, {scratch, 4, rows * cache->kv_heads * most, {}}),
             "%s: selected must not share memory with q, the cache, the table, lengths or scratch", what);
  SelectParams P{};
  P.c = *cache;
  P.q = q; P.q_token = q_token; P.q_head = q_head;
  P.table = table; P.table_row = table_row; P.table_pages = (int)table_pages;
  P.page_shift = __builtin_ctzll(cache->page_size);
  P.lengths = lengths;
  P.max_length = (int)(max_length < table_pages * cache->page_size ? max_length : table_pages * cache->page_size);
  P.per_kv = (int)(heads / cache->kv_heads); P.first = (int)first_pages; P.last = (int)last_pages;
  P.count = (int)selected_count;
  P.keys = reinterpret_cast<uint32_t*>(scratch); P.keys_row = most; P.selected = selected;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (most > selected_count) {             // (otherwise every page is kept)
    if (cache->dtype == TT_F16) launch_score<f16_t>(P, most, rows, st);
    else launch_score<bf16_t>(P, most, rows, st);
    const int err = check_launch(what);
    if (err) return err;
  }
  const dim3 pairs((unsigned)cache->kv_heads, (unsigned)rows);
  if (most <= 256 * 8) hipLaunchKernelGGL((page_pick_kernel<256, 8>), pairs, dim3(256), 0, st, P);
  else hipLaunchKernelGGL((page_pick_kernel<1024, 8>), pairs, dim3(1024), 0, st, P);
  return check_launch(what);
}
