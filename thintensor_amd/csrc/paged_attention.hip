// Attention over the paged cache.
#include "paged.h"
#include "tt_common.h"

namespace tt {

struct PagedParams {
  tt_paged_cache c;
  const void* q;
  int64_t q_token, q_head;
  const int32_t* table;
  int64_t table_row;
  int table_pages, page_shift;
  const int32_t* lengths;
  RowTokens of;
  const int32_t* selected;
  int selected_count;
  int heads, per_kv, window, shared, max_length;     // shared: tokens
  float scale_log2;                                  // scale * log2(e)
  const void* sinks;
  int sink_dtype;
  void* out;
  int64_t out_token, out_head;
};

__device__ __forceinline__ float sink_log2(const PagedParams& P, int h) {
  const float v = P.sink_dtype == TT_F32    ? reinterpret_cast<const float*>(P.sinks)[h]
                  : P.sink_dtype == TT_BF16 ? to_f32(reinterpret_cast<const bf16_t*>(P.sinks)[h])
                                            : to_f32(reinterpret_cast<const f16_t*>(P.sinks)[h]);
  return v * 0x1.715476p+0f;
}

// One workgroup takes one query head of one token, 256 tokens of its context at a time.
template <typename T>
__global__ __launch_bounds__(256) void paged_simple_kernel(PagedParams P) {
  const int token = blockIdx.x, head = blockIdx.y, dim = (int)P.c.head_dim, page = 1 << P.page_shift;
  __shared__ float q_s[256], p_s[256], red[4];
  __shared__ int id_s[256];
  const int row = P.of.cu ? P.of.find(token, 1, 1, 0) : token / P.of.each;
  int first;
  const int n_row = P.of.count(row, &first);
  if (token < first || token >= first + n_row) return;
  const int n = min(max(P.lengths[row], 0), P.max_length);
  const int hi = n - (n_row - 1 - (token - first)), lo = P.window > 0 ? max(0, hi - P.window) : 0;
  const int kvh = head / P.per_kv, tid = threadIdx.x;
  const T* q = reinterpret_cast<const T*>(P.q) + token * P.q_token + head * P.q_head;
  if (tid < dim) q_s[tid] = to_f32(q[tid]);
  __syncthreads();
  const float ninf = __builtin_bit_cast(float, 0xff800000u);
  float m = ninf, l = 0.0f, o = 0.0f;
  bool any = false;
  const int end = P.selected ? P.selected_count << P.page_shift : max(hi, 0);
  for (int u0 = P.selected ? 0 : lo; u0 < end; u0 += 256) {
    const int u = u0 + tid;
    int t = -1, id = -1;
    if (u < end) {
      const int logical = P.selected ? P.selected[((int64_t)row * P.c.kv_heads + kvh) * P.selected_count + (u >> P.page_shift)]
                                     : u >> P.page_shift;
      if (logical >= 0 && logical < P.table_pages) {
        t = (logical << P.page_shift) + (u & (page - 1));
        const int32_t* tab = t < P.shared ? P.table : P.table + row * P.table_row;
        id = tab[logical];
      }
    }
    const bool seen = t >= lo && t < hi;
    float s = ninf;
    if (seen) {
      if (id >= 0 && id < P.c.pages) {
        const T* k = reinterpret_cast<const T*>(P.c.k_pages) + (int64_t)id * P.c.k_page + kvh * P.c.k_head + (t & (page - 1)) * P.c.k_token;
        float dot = 0.0f;
        for (int d = 0; d < dim; d++) dot = __builtin_fmaf(q_s[d], to_f32(k[d]), dot);
        s = dot * P.scale_log2;
      } else {
        s = __builtin_bit_cast(float, 0x7fc00000u);
        id = 0;
      }
    }
    any = __syncthreads_or(seen) || any;
    float top = s;
#define TT_LEVEL(X) top = fmaxf(top, xor_partner<X>(top));
    TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float m_new = fmaxf(m, top), base = m_new == ninf ? 0.0f : m_new;
    const float a = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base);
    m = m_new;
    __syncthreads();
    p_s[tid] = p;
    id_s[tid] = seen ? id : -1;
    l = l * a + block_sum256(p, red);
    if (tid < dim) {
      o *= a;
      for (int i = 0; i < 256; i++) {
        if (id_s[i] < 0) continue;
        const int slot = (u0 + i) & (page - 1);
        o = __builtin_fmaf(p_s[i], to_f32(reinterpret_cast<const T*>(P.c.v_pages)[(int64_t)id_s[i] * P.c.v_page + kvh * P.c.v_head + slot * P.c.v_token + tid]), o);
      }
    }
    __syncthreads();
  }
  if (tid >= dim) return;
  T* out = reinterpret_cast<T*>(P.out) + token * P.out_token + head * P.out_head + tid;
  float r = 0.0f;
  if (any) {
    if (P.sinks) {
      const float sk = sink_log2(P, head), top = fmaxf(m, sk), e = __builtin_amdgcn_exp2f(m - top);
      r = o * e / (l * e + __builtin_amdgcn_exp2f(sk - top));
    } else {
      r = o / l;
    }
  }
  store<T>(out, r);
}

static int check_attention(const tt_paged_cache* c, int64_t table_pages, bool ragged, int64_t rows, int64_t tokens,
                           int64_t heads, int64_t window, int64_t shared_pages, int64_t selected_count, int64_t max_length,
                           const char* what) {
  const int rc = check_rows(c, table_pages, ragged, rows, tokens, heads, what);
  if (rc) return rc;
  TT_REQUIRE(heads > 0, "%s: heads must be a multiple of kv_heads", what);
  TT_REQUIRE(window >= 0 && max_length > 0, "%s: window must not be negative, max_length at least 1", what);
  TT_REQUIRE(shared_pages >= 0 && shared_pages <= table_pages, "%s: shared_pages outside the table", what);
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
  return 0;
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
  (void)scratch; (void)scratch_floats;
  PagedParams P{};
  P.c = *cache;
  P.q = q; P.q_token = q_token; P.q_head = q_head;
  P.table = table; P.table_row = table_row; P.table_pages = (int)table_pages;
  P.page_shift = __builtin_ctzll(cache->page_size);
  P.lengths = lengths;
  P.of = RowTokens{cu_tokens, (int)rows, (int)tokens, cu_tokens ? 0 : (int)(tokens / rows)};
  P.selected = selected; P.selected_count = (int)selected_count;
  P.heads = (int)heads; P.per_kv = (int)(heads / cache->kv_heads);
  const int64_t holds = table_pages * cache->page_size;
  P.max_length = (int)(max_length < holds ? max_length : holds);
  P.window = (int)(window < holds ? window : 0);
  P.shared = (int)(shared_pages * cache->page_size);
  P.scale_log2 = (float)((double)scale * 1.4426950408889634);
  P.sinks = sinks; P.sink_dtype = sink_dtype;
  P.out = out; P.out_token = out_token; P.out_head = out_head;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)tokens, (unsigned)heads);
  if (cache->dtype == TT_F16) hipLaunchKernelGGL((paged_simple_kernel<f16_t>), grid, dim3(256), 0, st, P);
  else hipLaunchKernelGGL((paged_simple_kernel<bf16_t>), grid, dim3(256), 0, st, P);
  return check_launch(what);
}
