// Appending to the paged cache with the rotation on the way.
#include "paged.h"
#include "tt_common.h"

namespace tt {

struct AppendParams {
  tt_paged_cache c;
  const void *q, *k, *v;
  void* q_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  const int32_t* table;
  int64_t table_row;
  int table_pages;
  const int32_t* starts;
  RowTokens of;
  int heads, rotary, interleaved;
  const double* inv_freq;
  float amplitude;
};

// One workgroup takes the tokens of one row that fall into one page.
template <typename T>
__global__ __launch_bounds__(256) void append_kernel(AppendParams P) {
  __shared__ float2 turn[128];
  const int page = (int)P.c.page_size, dim = (int)P.c.head_dim, kvh = (int)P.c.kv_heads, half = P.rotary >> 1;
  const int row = P.of.find(blockIdx.x, 1, page, 2);
  int first;
  const int n = P.of.count(row, &first);
  const int64_t start = P.starts[row];
  const int64_t unit = (int64_t)blockIdx.x - (first / page + 2 * row);
  // floor(start / page), negative positions too
  const int64_t logical = (start >> __builtin_ctz(page)) + unit;
  const int from = (int)max((int64_t)0, logical * page - start), to = (int)min((int64_t)n, (logical + 1) * page - start);
  if (from >= to) return;
  const int32_t id = logical >= 0 && logical < P.table_pages ? P.table[row * P.table_row + logical] : -1;
  const bool place = id >= 0 && id < P.c.pages;
  T* kp = reinterpret_cast<T*>(P.c.k_pages) + (int64_t)id * P.c.k_page;
  T* vp = reinterpret_cast<T*>(P.c.v_pages) + (int64_t)id * P.c.v_page;
  for (int i = from; i < to; i++) {
    const int64_t token = first + i, pos = start + i;
    const int slot = (int)(pos - logical * page);
    __syncthreads();
    for (int e = threadIdx.x; e < half; e += 256) {
      const double t = (double)pos * P.inv_freq[e] * 0.15915494309189533577;
      float s, c;
      sincospif(2.0f * (float)(t - __builtin_rint(t)), &s, &c);
      turn[e] = make_float2(c * P.amplitude, s * P.amplitude);
    }
    __syncthreads();
    const int units = dim - half;
    for (int u = threadIdx.x; u < (P.heads + kvh) * units; u += 256) {
      const int h = u / units, e = u - h * units;
      const bool is_k = h >= P.heads;
      const T* x = is_k ? reinterpret_cast<const T*>(P.k) + token * P.k_token + (h - P.heads) * P.k_head
                        : reinterpret_cast<const T*>(P.q) + token * P.q_token + h * P.q_head;
      if (is_k && !place) continue;
      T* o = is_k ? kp + (h - P.heads) * P.c.k_head + slot * P.c.k_token
                  : reinterpret_cast<T*>(P.q_out) + token * P.o_token + h * P.o_head;
      if (e < half) {
        const int ia = P.interleaved ? 2 * e : e, ib = P.interleaved ? 2 * e + 1 : e + half;
        const float a = to_f32(x[ia]), b = to_f32(x[ib]);
        const float2 cs = turn[e];
        store<T>(o + ia, a * cs.x - b * cs.y);
        store<T>(o + ib, b * cs.x + a * cs.y);
      } else {
        o[half + e] = x[half + e];
      }
    }
    if (place)
      for (int u = threadIdx.x; u < kvh * dim; u += 256) {
        const int h = u / dim, d = u - h * dim;
        vp[h * P.c.v_head + slot * P.c.v_token + d] = reinterpret_cast<const T*>(P.v)[token * P.v_token + h * P.v_head + d];
      }
  }
  if (!place || P.c.k_bounds == nullptr) return;
  __syncthreads();
  T* bp = reinterpret_cast<T*>(P.c.k_bounds) + (int64_t)id * P.c.b_page;
  const int slot0 = (int)(start + from - logical * page);
  for (int u = threadIdx.x; u < kvh * dim; u += 256) {
    const int h = u / dim, d = u - h * dim;
    T* b = bp + h * P.c.b_head + d;
    const T* x = kp + h * P.c.k_head + d;
    float lo = slot0 == 0 ? to_f32(x[0]) : to_f32(b[0]), hi = slot0 == 0 ? lo : to_f32(b[dim]);
    for (int s = slot0; s < slot0 + to - from; s++) {
      const float y = to_f32(x[s * P.c.k_token]);
      lo = y < lo || y != y ? y : lo;
      hi = y > hi || y != y ? y : hi;
    }
    store<T>(b, lo);
    store<T>(b + dim, hi);
  }
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_paged_cache_size(void) { return (int64_t)sizeof(tt_paged_cache); }

extern "C" int tt_rotary_append_paged(const tt_paged_cache* cache, const void* q, int64_t q_token, int64_t q_head,
                                      const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                                      int64_t v_head, const int32_t* table, int64_t table_row, int64_t table_pages,
                                      const int32_t* starts, const int32_t* cu_tokens, int64_t rows, int64_t tokens,
                                      int64_t heads, const double* inv_freq, int64_t rotary, int interleaved,
                                      float amplitude, void* q_out, int64_t qo_token, int64_t qo_head, void* stream) {
  const char* what = "rotary_append_paged";
  const int rc = check_rows(cache, table_pages, cu_tokens != nullptr, rows, tokens, 0, what);
  if (rc) return rc;
  TT_REQUIRE(heads >= 0 && heads <= 65535, "%s: bad head counts", what);
  TT_REQUIRE(rotary >= 0 && rotary <= cache->head_dim && rotary % 2 == 0, "%s: rotary dims must be even and at most head_dim", what);
  if (rows == 0 || tokens == 0) return TT_OK;
  TT_REQUIRE(k && v && table && starts && (heads == 0 || (q && q_out)) && (rotary == 0 || inv_freq), "%s: null pointer", what);
  const int64_t dim = cache->head_dim, kvh = cache->kv_heads;
  const Region qr(q, 2, dim, {{tokens, q_token}, {heads, q_head}}), kr(k, 2, dim, {{tokens, k_token}, {kvh, k_head}}),
      vr(v, 2, dim, {{tokens, v_token}, {kvh, v_head}}), made(q_out, 2, dim, {{tokens, qo_token}, {heads, qo_head}});
  const PagedRegions held(cache);
  TT_REQUIRE(held.once(), "%s: pages, heads, tokens and arrays of the cache must not share memory", what);
  TT_REQUIRE(held.apart_from(qr) && held.apart_from(kr) && held.apart_from(vr) && held.apart_from(made),
             "%s: the cache must not share memory with q, k, v or q_out", what);
  TT_REQUIRE(made.once() && (made.same(qr) || apart(made, qr)) && apart(made, kr) && apart(made, vr),
             "%s: q_out may be q, but must not share memory with itself, k, v or q otherwise", what);
  AppendParams P{};
  P.c = *cache;
  P.q = q; P.k = k; P.v = v; P.q_out = q_out;
  P.q_token = q_token; P.q_head = q_head; P.k_token = k_token; P.k_head = k_head;
  P.v_token = v_token; P.v_head = v_head; P.o_token = qo_token; P.o_head = qo_head;
  P.table = table; P.table_row = table_row; P.table_pages = (int)table_pages; P.starts = starts;
  P.of = RowTokens{cu_tokens, (int)rows, (int)tokens, cu_tokens ? 0 : (int)(tokens / rows)};
  P.heads = (int)heads; P.rotary = (int)rotary; P.interleaved = interleaved != 0;
  P.inv_freq = inv_freq; P.amplitude = amplitude;
  const dim3 grid((unsigned)(tokens / cache->page_size + 2 * rows));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cache->dtype == TT_F16) hipLaunchKernelGGL((append_kernel<f16_t>), grid, dim3(256), 0, st, P);
  else hipLaunchKernelGGL((append_kernel<bf16_t>), grid, dim3(256), 0, st, P);
  return check_launch(what);
}
