// Attention over the paged cache: the plan of a call, its checks, and the join of its parts.
#include "paged_attention.h"

namespace tt {

// Joins the parts of one (token, head).  Every wave forms all weights; sixteen bytes of a part's sum per
// thread, the parts dealt over the threads' rows and joined in LDS.  A part without weight is not read,
// nor does its maximum count.
template <typename T, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(PagedParams P) {
  constexpr int PIECES = D / 4, ROWS = THREADS / PIECES;
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 63;
  const int piece = threadIdx.x % PIECES, r = threadIdx.x / PIECES;
  __shared__ float e_s[kMostParts];
  __shared__ __attribute__((aligned(16))) f4_t sum[ROWS][PIECES];
  const int64_t at = ((int64_t)token * P.heads + head) * P.parts;
  const float2* ml = P.part_ml + at;
  const f4_t* po = reinterpret_cast<const f4_t*>(P.part_o + at * D);
  if (P.of.cu) {                                       // tokens behind the last row are left as they were
    const int row = P.of.find(token, 1, 1, 0);
    int first;
    const int n = P.of.count(row, &first);
    if (token < first || token >= first + n) return;
  }
  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  float M = ninf;
  for (int k = lane; k < P.parts; k += 64) {
    const float2 v = ml[k];
    if (v.y != 0.0f) M = fmaxf(M, v.x);                // (NaN counts)
  }
#define TT_LEVEL(X) M = fmaxf(M, xor_partner<X>(M));
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
  const float base = M == ninf ? 0.0f : M;
  float l = 0.0f;
  for (int k = lane; k < P.parts; k += 64) {
    const float2 v = ml[k];
    const float e = v.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(v.x - base);
    l = __builtin_fmaf(v.y, e, l);
    if (threadIdx.x < 64) e_s[k] = v.y == 0.0f ? -1.0f : e;
  }
  l = xor_sum(l, 1, 64);
  __syncthreads();
  f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int MORE = 8;
  for (int i = r; i < P.parts; i += MORE * ROWS) {
    f4_t more[MORE];
    float e[MORE];
#pragma unroll
    for (int k = 0; k < MORE; k++) {
      const int p = i + k * ROWS;
      e[k] = p < P.parts ? e_s[p] : -1.0f;
      if (!(e[k] < 0.0f)) more[k] = po[(int64_t)p * PIECES + piece];
    }
#pragma unroll
    for (int k = 0; k < MORE; k++)
      if (!(e[k] < 0.0f)) acc += more[k] * e[k];
  }
  sum[r][piece] = acc;
  __syncthreads();
  if (r != 0) return;
#pragma unroll
  for (int k = 1; k < ROWS; k++) acc += sum[k][piece];
  const float f = finish_scale(P, head, M, l);
  if (l == 0.0f) acc = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
  store_four<T>(reinterpret_cast<T*>(P.out) + token * P.out_token + head * P.out_head + 4 * piece, acc * f, P.out_vec);
}

template <typename T, int D>
static int launch_join(const PagedParams& P, hipStream_t st, const char* what) {
  const dim3 grid((unsigned)P.of.tokens, (unsigned)P.heads);
  if ((int64_t)P.heads * P.of.tokens > 4 * device_cus()) hipLaunchKernelGGL((paged_join_kernel<T, D, 64>), grid, dim3(64), 0, st, P);
  else hipLaunchKernelGGL((paged_join_kernel<T, D, 256>), grid, dim3(256), 0, st, P);
  return check_launch(what);
}
template <typename T>
static int launch_join(const PagedParams& P, hipStream_t st, const char* what) {
  if (P.c.head_dim == 64) return launch_join<T, 64>(P, st, what);
  if (P.c.head_dim == 128) return launch_join<T, 128>(P, st, what);
  return launch_join<T, 256>(P, st, what);
}

// One of a call's launches.
struct PagedJob {
  bool many;
  int waves;                            // many: of a workgroup, 32 columns each
  int blocks16, row_tiles, rows;        // few: columns of a workgroup in sixteens, workgroups of a row, rows
  int64_t tiles;                        // many: column tiles
  int splits, share, wide;
};

struct PagedPlan {
  int64_t limit, shared, window;        // tokens
  PagedJob own, prefix;
  int parts;
};

// Workgroups that share a row's tokens, for `groups` of them that each may take up to `tiles` tiles of 32.  A
// workgroup alone saves the join (3.7 us in a row of calls).  With a CU for each, eight waves instead of four have more on
// its way (one row of 8 KV heads in a graph, us: x 64, 256 tokens 5.1 and 5.4, 512 7.0 and 6.1, 768 9.0 and 7.4, shared 8.6;
// x 128, 256 tokens 6.9 and 6.6, 512 9.6 and 7.8, 768 12.3 and 9.6, shared 10.0).  Where rows are split, few and long
// workgroups are best, two for each CU, or three for every four CUs where the rows alone are few: parts cost their sums,
// short workgroups their start (us with 12, 4 and 2 a CU: 16 rows of 4001 tokens, 40 / 10 heads x 128, 75, 68 and 64, 64 rows
// to 8001, 16 / 2 x 256, 167, 137 and 139; with 2, 1 and 3/4 a CU: one row of 120000, 64 / 8 x 128, 94.8, 92.2 and 90.4).
// Lengths are on the device, so where a bound leaves room for rows much longer than others (past 8192 tokens) rows are
// cut finer, and by 8192 tokens at the least while that is no more than 32 workgroups a CU (64 rows, 64 / 8 x 128: one of 65536 tokens among 500s 192 us, 642 with two
// workgroups a CU; all of 500 30.7 and 24.6).  Rows of like length lose little to it where tables are wider than they need
// (32 rows of 4001 to 8001 tokens, 64 / 8 x 128, bound at 8192, 8256, 32768 and 131072: 154, 162, 156 and 152 us in 2, 12, 12 and
// 16 parts; 4000 tokens each, bound at 4032 and 32768, 98 and 100).  `cached`: at x 64, where rows read the same pages for themselves,
// which come from the caches, a CU's own pace decides (eight rows of 16 columns behind 16384 tokens, 32 / 8 heads: 28 us with
// two workgroups a CU, 43 with 3/4; wider heads and more rows are not slower by the rule above).
static void split_few(int64_t groups, int64_t tiles, bool parts, bool cached, PagedJob* j) {
  const int64_t cus = device_cus();
  j->splits = 1;
  j->share = (int)tiles;
  j->wide = !parts && groups <= cus && tiles > 8;
  if (!parts && (tiles <= 24 || (groups >= cus && tiles <= 64))) return;
  j->wide = 0;
  const bool uneven = !parts && tiles > 256;
  const int64_t want = groups < cus / 2 ? (cached ? 2 * cus : 3 * cus / 4) : uneven ? 12 * cus : 2 * cus;
  int64_t share = (tiles * groups + want - 1) / want;
  if (share < 8) share = 8;
  const int64_t finest = (tiles * groups + 32 * cus - 1) / (32 * cus);      // (most of these workgroups find nothing to do)
  if (uneven && share > 256) share = finest > 256 ? finest : 256;
  if (share < (tiles + 511) / 512) share = (tiles + 511) / 512;
  if (share > tiles) share = tiles;                      // (rows enough for one part each ask for any share)
  j->share = (int)share;
  j->splits = (int)((tiles + share - 1) / share);        // (a short last one fills what the others leave)
  if (j->splits < 1) j->splits = 1;
}

// Waves of a workgroup, 32 columns each, for rows of `cols` columns, `groups` of them times KV heads.  Eight share what
// comes to LDS further, and a split prefix fills the card with either (4096 queries behind 16384 tokens, 64 / 8 heads: x 128
// 2212 us with four, 2075 with eight; 512 columns behind 32768 shared tokens 143 and 140; x 256, with registers for one wave
// of a SIMD or two, 1957 and 1109 us for 2048 behind 8192).  Four lose less to the ends of rows and, at x 64 with its three
// workgroups of four on a CU, spread over the CUs better until there are four workgroups of eight for each (64 / 8 heads x 64,
// 1027 tokens of 4099: 107 us with four, 126 with eight, a window of 2048 70 and 81, 4096 tokens 197 and 188; x 128, 40 / 10
// heads, eight rows of 100 tokens and less 67 and 79, four of 512 and less 143 and 130).
static int many_waves(int64_t head_dim, int64_t cols, int64_t groups) {
  if (head_dim == 256) return 8;
  return head_dim == 128 ? (cols > 256 ? 8 : 4) : cols > 128 && groups * ((cols + 255) / 256) >= 4 * device_cus() ? 8 : 4;
}

// Workgroups of them that a CU holds (registers, LDS).
static int many_per_cu(int64_t head_dim, int waves) { return waves == 8 ? (head_dim == 64 ? 2 : 1) : (head_dim == 64 ? 3 : 2); }

// Workgroups that share a column tile's tokens, enough to fill the card, with at least six tiles each: a part costs the
// write and the reading of its sums, and the join its launch (one row of 512 tokens, 40 heads of 128: 32.3 us in two parts of
// four tiles, 24.7 in one; 512 behind 4096 70.5 with at least four tiles, 66.8 with six, 65.8 with eight; 49 rows of eight
// heads behind 30496 shared tokens 40.8, 42.6 and 45.7).  Lengths are on the device, so one long row among short ones is one
// workgroup a KV head where the tiles of all rows fill the card: seven single tokens behind 65536 beside a chunk of 512 of
// another row, 64 / 8 x 128, take 1871 us, as two calls 321 and 26.
static void split_many(int64_t groups, int64_t tiles, int per_cu, PagedJob* j) {
  const int64_t most = tiles / 6, fill = per_cu * device_cus() / (groups > 0 ? groups : 1);
  int64_t s = most < fill ? most : fill;
  s = s < 1 ? 1 : s > 256 ? 256 : s;
  j->splits = (int)s;
  j->share = 1;
}

// Whether the rows' own pages go to the kernel for many columns.  That for few takes a row's columns in blocks, each with all
// of the row's tokens; it starts sooner and costs less per workgroup, so what decides is the K and V that all its blocks
// would read, in MB, and their number.  us of few and many (8, 10, 2 KV heads at x 64, 128, 256):
//   x 64, blocks of 64: 64 columns behind 1024 tokens, 4 rows 13.9 and 15.9 (8 MB), 16 rows 26.5 and 23.2 (33); 128 behind
//     4096 17.2 and 17.4 (17), 256 behind 4096 25.3 and 20.7 (33)
//   x 128, of 32: 128 behind 1024 14.4 and 20.6 (21), behind 4096 30.1 and 24.8 (84); 64 behind 4096 21.0 and 23.0 (42)
//   x 256, of 16: 64 behind 4096 18.3 and 28.6 (67), 128 31.3 and 31.4 (134), 512 60.8 and 37.8 (537)
// One block of a row reads no more than the row has to: with less than half of the CUs taken, or half a block, it stays
// ahead at any length (x 64, 4 rows of 64 behind 16384: 34.3 and 37.9; x 128, 16 columns of 16 rows behind 4096: 84 and 79,
// 32 columns 100 and 82).  Many short blocks queue (x 128, 16 rows of 160 columns, 16 tokens each: 21.8 and 12.9).
// Rows of unequal counts get blocks for all tokens each, most without columns.
static bool own_by_many(const tt_paged_cache* c, bool ragged, int64_t rows, int64_t tokens, int64_t G, int64_t reach) {
  const int64_t D = c->head_dim, width = few_columns(D), cols = (ragged ? tokens : tokens / rows) * G, cus = device_cus();
  const int64_t blocks = (cols + width - 1) / width;
  if (!ragged && blocks == 1 && (2 * cols <= width || D == 256 || 2 * rows * c->kv_heads < cus)) return false;
  if (rows * blocks * c->kv_heads > (ragged && D != 256 ? cus : 2 * cus)) return true;
  return 4e-6 * reach * c->kv_heads * D * (ragged ? rows + blocks : rows * blocks) > (D == 64 ? 20 : D == 128 ? 50 : 140);
}

// Who computes the shared pages once for all rows: nobody (every row for itself, from row 0's pages, most of which then
// come from the caches), the kernel for few columns in blocks, in one launch with the rows' own pages, or that for many in
// a launch before it.  Times are estimated from the MB that a row shares: what a row or a block of sixteen columns costs
// for each, what a column costs in the kernel for many, and what each way costs to begin with (less where the rows alone
// would be split and joined too).  us of nobody, few, many in a row of calls:
//   x 64, 8 KV heads: 16 rows of 4 columns behind 1024 tokens (2 MB) 11.0, 14.1 and 18.4, behind 16384 (34 MB) 41.9,
//     21.8 and 26.6; 64 rows of 16 behind 4096 (8 MB) 46.0, 49.9 and 40.9, behind 16384 116.6, 94.7 and 67.0
//   x 128, 10: 8 rows of 4 behind 1024 (5 MB) 12.3, 13.6 and 23.2, behind 4096 23.6, 15.2 and 25.7; 32 rows behind 4096 (21
//     MB) 55.0, 33.6 and 33.7, behind 16384 150, 70 and 45
//   x 256, 2: 32 rows of 8 behind 1024 (4 MB) 22.3, 17.9 and 37.7, behind 16384 80, 64 and 62
// Rows that go to the kernel for many columns by themselves have their matrix products in any case; sharing saves them
// the padding of their column tiles (16 rows of 80 columns, x 128, 8 KV heads, behind 16384 tokens: 175 us by themselves, 123
// shared; behind 4096 60 and 57; 16 rows of 128 columns, x 64, 64 and 73).
enum SharedBy { kNobody, kFew, kMany };
static SharedBy shared_by(const tt_paged_cache* c, bool own_many, bool ragged, int64_t rows, int64_t tokens, int64_t G,
                          int64_t window, int64_t reach) {
  const int64_t D = c->head_dim, cols = tokens * G, each = tokens / rows;
  if (window > 0 && window + each < reach) reach = window + each;
  const double mb = 4e-6 * reach * c->kv_heads * D;
  if (own_many) {
    const int64_t mc = 32 * many_waves(D, each * G, rows * c->kv_heads), padded = ragged ? cols + rows * mc / 2 : rows * ((each * G + mc - 1) / mc * mc);
    return 8 + 0.1 * D + mb * (0.2 + 0.001 * cols) < mb * (0.2 + 0.001 * padded) ? kMany : kNobody;
  }
  const int64_t tiles = (reach + 31) / 32;
  const bool parts = tiles > (rows * c->kv_heads >= device_cus() ? 64 : 24);
  const double none = mb * (0.25 + 0.05 * (ragged ? (cols + 8 * rows) / 16.0 : rows * ((each * G + 15) / 16)));
  const double few = (parts ? 2 : 6) + mb * (0.25 + 0.05 * ((cols + 15) / 16));
  const double many = (parts ? 13 : 16) + mb * (0.2 + 0.001 * cols);
  return none <= few && none <= many ? kNobody : few <= many ? kFew : kMany;
}

static PagedPlan plan(const tt_paged_cache* c, int64_t table_pages, bool ragged, int64_t rows, int64_t tokens, int64_t heads,
                      int64_t window, int64_t shared_pages, int64_t selected_count, int64_t max_length) {
  PagedPlan p{};
  const int64_t holds = table_pages * c->page_size, G = heads / c->kv_heads;
  p.limit = max_length < holds ? max_length : holds;
  p.window = window < p.limit ? window : 0;
  const int64_t each = ragged ? 0 : tokens / rows;
  const int tt = many_tile_tokens(c->head_dim), few = few_columns(c->head_dim);
  const auto blocks16 = [&](int64_t cols) { return cols <= 16 || few == 16 ? 1 : cols <= 32 || few == 32 ? 2 : 4; };
  int64_t reach = p.limit;
  if (p.window > 0 && p.window + (ragged ? tokens : each) < reach) reach = p.window + (ragged ? tokens : each);
  p.own.many = selected_count == 0 && own_by_many(c, ragged, rows, tokens, G, reach);
  const int64_t cols = tokens * G, prefix = shared_pages * c->page_size, reach_shared = prefix < p.limit ? prefix : p.limit;
  const SharedBy by = rows > 1 && shared_pages > 0 ? shared_by(c, p.own.many, ragged, rows, tokens, G, p.window, reach_shared) : kNobody;
  p.shared = by == kNobody ? 0 : prefix;
  if (by == kMany) {
    p.prefix.many = true;
    p.prefix.waves = c->head_dim == 256 || cols > 128 ? 8 : 4;
    const int mc = 32 * p.prefix.waves;
    p.prefix.tiles = (cols + mc - 1) / mc;
    split_many(p.prefix.tiles * c->kv_heads, (reach_shared + tt - 1) / tt, many_per_cu(c->head_dim, p.prefix.waves), &p.prefix);
  } else if (by == kFew) {
    p.prefix.blocks16 = 4e-6 * reach_shared * c->kv_heads * c->head_dim < 8 ? 1 : blocks16(cols < 32 ? cols : 32);
    p.prefix.row_tiles = (int)((cols + 16 * p.prefix.blocks16 - 1) / (16 * p.prefix.blocks16));
    p.prefix.rows = 1;
    split_few(c->kv_heads * p.prefix.row_tiles, (reach_shared + 31) / 32, true, false, &p.prefix);
  }
  // tokens of its own that a row's queries may see
  reach = p.limit > p.shared ? p.limit - p.shared : 0;
  if (p.window > 0 && p.window + (ragged ? tokens : each) < reach) reach = p.window + (ragged ? tokens : each);
  if (selected_count > 0) {
    const int64_t pages = (p.limit - 1) / c->page_size + 1;
    reach = (selected_count < pages ? selected_count : pages) * c->page_size;
  }
  if (p.own.many) {
    p.own.waves = many_waves(c->head_dim, tokens / rows * G, rows * c->kv_heads);
    const int mc = 32 * p.own.waves;
    if (p.window > 0 && p.window + mc / G + 1 < reach) reach = p.window + mc / G + 1;      // of a column tile
    p.own.row_tiles = (int)((each * G + mc - 1) / mc);
    p.own.tiles = ragged ? tokens * G / mc + rows : rows * p.own.row_tiles;
    split_many(p.own.tiles * c->kv_heads, (reach + tt - 1) / tt + 1, many_per_cu(c->head_dim, p.own.waves), &p.own);
  } else {
    const int64_t most = ragged ? cols : each * G;
    p.own.blocks16 = by == kFew ? p.prefix.blocks16 : blocks16(most);      // (one kernel for both)
    p.own.row_tiles = (int)((most + 16 * p.own.blocks16 - 1) / (16 * p.own.blocks16));
    p.own.rows = (int)rows;
    // (one tile more where they may begin inside one)
    split_few(rows * c->kv_heads, (reach + 31) / 32 + (p.window > 0 || p.shared % 32 != 0 ? 1 : 0), false,
              c->head_dim == 64 && shared_pages > 0 && p.shared == 0, &p.own);
    // a selection may name its pages anywhere in it
    const int64_t listed = (selected_count * c->page_size + 31) / 32;
    if (listed > p.own.splits * p.own.share) p.own.share = (int)((listed + p.own.splits - 1) / p.own.splits);
  }
  p.parts = p.own.splits + (p.shared > 0 ? p.prefix.splits : 0);
  return p;
}

static int64_t scratch_floats_of(const PagedPlan& p, const tt_paged_cache* c, int64_t tokens, int64_t heads) {
  return p.parts == 1 ? 0 : tokens * heads * p.parts * (c->head_dim + 2);
}

static int launch_many(PagedParams P, const PagedJob& j, bool shared, int part0, hipStream_t st, const char* what) {
  P.shared_job = shared;
  P.part0 = part0;
  P.share = j.share;
  P.row_tiles = j.row_tiles;
  P.tiles = (int)j.tiles;
  // in order of their length where they do not all run at once
  P.ordered = !shared && P.window == 0 && P.of.rows <= 64 && j.tiles * P.c.kv_heads * j.splits > many_per_cu(P.c.head_dim, j.waves) * device_cus();
  return launch_paged_many(P, j.waves, j.splits, st, what);
}

static FewJob few_job(const PagedParams& P, const PagedJob& j, int part0) {
  return FewJob{(int)(P.c.kv_heads * j.row_tiles * j.rows * j.splits), j.row_tiles, j.rows, j.share, part0};
}

static int check_attention(const tt_paged_cache* c, int64_t table_pages, bool ragged, int64_t rows, int64_t tokens,
                           int64_t heads, int64_t window, int64_t shared_pages, int64_t selected_count, int64_t max_length,
                           const char* what) {
  const int rc = check_rows(c, table_pages, ragged, rows, tokens, heads, what);
  if (rc) return rc;
  TT_REQUIRE(heads > 0, "%s: heads must be a multiple of kv_heads", what);
  TT_REQUIRE(window >= 0 && max_length >= (rows > 0), "%s: window must not be negative, max_length at least 1", what);
  TT_REQUIRE(shared_pages >= 0 && shared_pages <= table_pages, "%s: shared_pages outside the table", what);
  TT_REQUIRE((tokens * heads) / 128 + rows * c->kv_heads < (1 << 23), "%s: too many queries for one call", what);
  TT_REQUIRE(selected_count >= 0 && selected_count <= 65536 && (selected_count == 0 || (!ragged && tokens == rows && shared_pages == 0)),
             "%s: selected pages (65536 at most) are for one query per row, without shared pages", what);
  return TT_OK;
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_gqa_attention_paged_scratch_floats(const tt_paged_cache* cache, int64_t table_pages, int ragged,
                                                         int64_t rows, int64_t tokens, int64_t heads, int64_t window,
                                                         int64_t shared_pages, int64_t selected_count, int64_t max_length) {
  const int rc = check_attention(cache, table_pages, ragged != 0, rows, tokens, heads, window, shared_pages, selected_count,
                                 max_length, "gqa_attention_paged");
  if (rc) return rc;
  if (rows == 0 || tokens == 0) return 0;
  const PagedPlan p = plan(cache, table_pages, ragged != 0, rows, tokens, heads, window, shared_pages, selected_count, max_length);
  return scratch_floats_of(p, cache, tokens, heads);
}

extern "C" int tt_gqa_attention_paged(const tt_paged_cache* cache, const void* q, int64_t q_token, int64_t q_head,
                                      const int32_t* table, int64_t table_row, int64_t table_pages, const int32_t* lengths,
                                      const int32_t* cu_tokens, int64_t rows, int64_t tokens, int64_t heads, int64_t window,
                                      int64_t shared_pages, const int32_t* selected, int64_t selected_count,
                                      int64_t max_length, const void* sinks, int sink_dtype, float scale, float* scratch,
                                      int64_t scratch_floats, void* out, int64_t out_token, int64_t out_head, void* stream) {
  const char* what = "gqa_attention_paged";
  if (selected == nullptr) selected_count = 0;
  const int rc = check_attention(cache, table_pages, cu_tokens != nullptr, rows, tokens, heads, window, shared_pages,
                                 selected_count, max_length, what);
  if (rc) return rc;
  TT_REQUIRE(selected == nullptr || selected_count > 0, "%s: selected without a count", what);
  TT_REQUIRE(sinks == nullptr || valid_out_dtype(sink_dtype), "%s: sinks must be fp16, bf16 or fp32", what);
  TT_REQUIRE(scale - scale == 0.0f, "%s: scale must be finite", what);
  if (rows == 0 || tokens == 0) return TT_OK;
  TT_REQUIRE(q && out && lengths && table, "%s: null pointer", what);
  const Region qr(q, 2, cache->head_dim, {{tokens, q_token}, {heads, q_head}});
  const Region made(out, 2, cache->head_dim, {{tokens, out_token}, {heads, out_head}});
  TT_REQUIRE(made.once() && (made.same(qr) || apart(made, qr)) && PagedRegions(cache).apart_from(made),
             "%s: out may be q, but must not share memory with itself, the cache or q otherwise", what);
  const PagedPlan p = plan(cache, table_pages, cu_tokens != nullptr, rows, tokens, heads, window, shared_pages, selected_count, max_length);
  const int64_t need = scratch_floats_of(p, cache, tokens, heads);
  TT_REQUIRE(need == 0 || (scratch && aligned(scratch, 16) && scratch_floats >= need), "%s: scratch too small or not 16-byte aligned", what);
  PagedParams P{};
  P.c = *cache;
  P.q = q; P.q_token = q_token; P.q_head = q_head;
  P.table = table; P.table_row = table_row; P.table_pages = (int)table_pages;
  P.page_shift = __builtin_ctzll(cache->page_size);
  P.lengths = lengths;
  P.of = RowTokens{cu_tokens, (int)rows, (int)tokens, cu_tokens ? 0 : (int)(tokens / rows)};
  P.selected = selected; P.selected_count = (int)selected_count;
  P.heads = (int)heads; P.per_kv = (int)(heads / cache->kv_heads);
  P.max_length = (int)p.limit; P.window = (int)p.window; P.shared = (int)p.shared;
  P.shared_entries = (int)shared_pages;
  P.q_vec = aligned(q, 16) && ((q_token | q_head) & 7) == 0;
  P.out_vec = aligned(out, 8) && ((out_token | out_head) & 3) == 0;
  P.scale_log2 = (float)((double)scale * 1.4426950408889634);
  P.sinks = sinks; P.sink_dtype = sink_dtype;
  P.out = out; P.out_token = out_token; P.out_head = out_head;
  hipStream_t st = static_cast<hipStream_t>(stream);
  P.parts = p.parts;
  P.part_o = scratch;
  P.part_ml = reinterpret_cast<float2*>(scratch + tokens * heads * p.parts * cache->head_dim);
  int err = TT_OK;
  if (p.shared > 0 && p.prefix.many) err = launch_many(P, p.prefix, true, p.own.splits, st, what);
  if (p.shared > 0 && !p.prefix.many) P.few[1] = few_job(P, p.prefix, p.own.splits);
  if (err == TT_OK && p.own.many) err = launch_many(P, p.own, false, 0, st, what);
  if (err == TT_OK && !p.own.many) {
    P.few[0] = few_job(P, p.own, 0);
    P.wide = p.own.wide;
    err = launch_paged_few(P, p.own.blocks16, st, what);
  }
  if (err != TT_OK || p.parts == 1) return err;
  return cache->dtype == TT_F16 ? launch_join<f16_t>(P, st, what) : launch_join<bf16_t>(P, st, what);
}
