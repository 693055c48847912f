// Selecting the pages that a query reads by the bounds of their keys.
#include "paged.h"
#include "tt_common.h"

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
  float* scores;
  int64_t scores_row;          // of one (row, KV head)
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

template <typename T>
__global__ __launch_bounds__(256) void page_score_kernel(SelectParams P) {
  const int row = blockIdx.z, kvh = blockIdx.y, dim = (int)P.c.head_dim;
  const int p = blockIdx.x * 256 + threadIdx.x;
  if (p >= row_pages(P, row)) return;
  const int32_t id = P.table[row * P.table_row + p];
  float best = __builtin_bit_cast(float, 0x7fc00000u);
  if (id >= 0 && id < P.c.pages) {
    const T* b = reinterpret_cast<const T*>(P.c.k_bounds) + (int64_t)id * P.c.b_page + kvh * P.c.b_head;
    best = __builtin_bit_cast(float, 0xff800000u);
    for (int g = 0; g < P.per_kv; g++) {
      const T* q = reinterpret_cast<const T*>(P.q) + row * P.q_token + (kvh * P.per_kv + g) * P.q_head;
      double sum = 0.0;
      for (int d = 0; d < dim; d++) {
        const double x = (double)to_f32(q[d]), lo = x * (double)to_f32(b[d]), hi = x * (double)to_f32(b[dim + d]);
        sum += lo > hi || lo != lo ? lo : hi;
      }
      const float s = (float)sum;
      best = s > best || s != s ? s : best;
    }
  }
  P.scores[((int64_t)row * P.c.kv_heads + kvh) * P.scores_row + p] = best;
}

// A page is kept where fewer than the free places go to better ones.
__global__ __launch_bounds__(256) void page_pick_kernel(SelectParams P) {
  const int row = blockIdx.y, kvh = blockIdx.x;
  const int64_t at = (int64_t)row * P.c.kv_heads + kvh;
  const float* s = P.scores + at * P.scores_row;
  int32_t* out = P.selected + at * P.count;
  const int pages = row_pages(P, row), first = min(P.first, pages), last = max(first, pages - P.last);
  const int places = P.count - (first + pages - last);
  __shared__ int base, part[4];
  if (threadIdx.x == 0) base = 0;
  for (int p0 = 0; p0 < pages; p0 += 256) {
    const int p = p0 + threadIdx.x;
    bool keep = p < pages && (p < first || p >= last);
    if (p < pages && !keep) {
      const uint32_t mine = score_key(s[p]);
      int better = 0;
      for (int o = first; o < last; o++) {
        const uint32_t k = score_key(s[o]);
        better += k > mine || (k == mine && o < p);
      }
      keep = better < places;
    }
    const uint64_t mask = __builtin_amdgcn_ballot_w64(keep);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) part[wave] = __popcll(mask);
    __syncthreads();
    int put = base;
    for (int w = 0; w < wave; w++) put += part[w];
    put += __popcll(mask & ((1ull << lane) - 1));
    if (keep) out[put] = p;
    __syncthreads();
    if (threadIdx.x == 0) base += part[0] + part[1] + part[2] + part[3];
    __syncthreads();
  }
  __syncthreads();
  for (int i = base + threadIdx.x; i < P.count; i += 256) out[i] = -1;
}

static int check_select(const tt_paged_cache* c, int64_t table_pages, int64_t rows, int64_t heads, int64_t max_length,
                        const char* what) {
  const int rc = check_rows(c, table_pages, false, rows, rows, heads, what);
  if (rc) return rc;
  TT_REQUIRE(c->k_bounds, "%s: the cache keeps no k_bounds", what);
  TT_REQUIRE(max_length > 0, "%s: max_length must be at least 1", what);
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
  SelectParams P{};
  P.c = *cache;
  P.q = q; P.q_token = q_token; P.q_head = q_head;
  P.table = table; P.table_row = table_row; P.table_pages = (int)table_pages;
  P.page_shift = __builtin_ctzll(cache->page_size);
  P.lengths = lengths;
  P.max_length = (int)(max_length < table_pages * cache->page_size ? max_length : table_pages * cache->page_size);
  P.per_kv = (int)(heads / cache->kv_heads); P.first = (int)first_pages; P.last = (int)last_pages;
  P.count = (int)selected_count;
  P.scores = scratch; P.scores_row = most; P.selected = selected;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((most + 255) / 256), (unsigned)cache->kv_heads, (unsigned)rows);
  if (cache->dtype == TT_F16) hipLaunchKernelGGL((page_score_kernel<f16_t>), grid, dim3(256), 0, st, P);
  else hipLaunchKernelGGL((page_score_kernel<bf16_t>), grid, dim3(256), 0, st, P);
  const int err = check_launch(what);
  if (err) return err;
  hipLaunchKernelGGL(page_pick_kernel, dim3((unsigned)cache->kv_heads, (unsigned)rows), dim3(256), 0, st, P);
  return check_launch(what);
}
