// The paged KV cache as the kernels see it, the rows' tokens and the checks of its descriptor
// (layout: tt_paged_cache in thintensor_hip.h).
#pragma once

#include "tt_abi_internal.h"
#include "tt_common.h"
#include "tt_regions.h"

namespace tt {

inline int check_paged(const tt_paged_cache* c, const char* what) {
  TT_REQUIRE(c != nullptr, "%s: null cache", what);
  TT_REQUIRE(c->k_pages && c->v_pages, "%s: null cache pointer", what);
  TT_REQUIRE(valid_act_dtype((int)c->dtype), "%s: the cache must be fp16 or bf16", what);
  TT_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim must be 64, 128 or 256", what);
  TT_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
             "%s: page_size must be 16, 32, 64, 128 or 256", what);
  TT_REQUIRE(c->pages > 0 && c->pages < (1LL << 31), "%s: bad number of pages", what);
  TT_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 65535, "%s: bad kv_heads", what);
  TT_REQUIRE(aligned(c->k_pages, 16) && aligned(c->v_pages, 16) && aligned(c->k_bounds, 16) &&
                 ((c->k_page | c->k_head | c->k_token | c->v_page | c->v_head | c->v_token | c->b_page | c->b_head) & 7) == 0,
             "%s: every vector of the cache must start on a 16-byte boundary", what);
  // a lane's places inside a page and head are unsigned 32-bit byte offsets
  const int64_t most = (1LL << 31) / 2 / c->page_size;
  TT_REQUIRE(c->k_token >= 0 && c->k_token < most && c->v_token >= 0 && c->v_token < most,
             "%s: tokens of a page must lie in order within 2 GiB", what);
  return TT_OK;
}

// The table (of no pages where there are no rows) and the rows' tokens: what every operator on pages takes.
inline int check_rows(const tt_paged_cache* c, int64_t table_pages, bool ragged, int64_t rows, int64_t tokens, int64_t heads,
                      const char* what) {
  const int rc = check_paged(c, what);
  if (rc) return rc;
  TT_REQUIRE(rows >= 0 && rows <= 65535, "%s: at most 65535 rows", what);
  TT_REQUIRE(tokens >= 0 && tokens <= (1 << 22), "%s: at most 2^22 tokens", what);
  TT_REQUIRE(ragged || tokens == 0 || (rows > 0 && tokens % rows == 0), "%s: tokens must divide over the rows", what);
  TT_REQUIRE(heads % c->kv_heads == 0 && heads <= 65535, "%s: heads must be a multiple of kv_heads (65535 at most)", what);
  TT_REQUIRE(table_pages >= (rows > 0) && table_pages * c->page_size < (1LL << 30), "%s: a row's pages must hold fewer than 2^30 tokens", what);
  return TT_OK;
}

// What the cache takes up: keys, values, bounds.
struct PagedRegions {
  Region of[3];
  PagedRegions(const tt_paged_cache* c)
      : of{{c->k_pages, 2, c->head_dim, {{c->pages, c->k_page}, {c->kv_heads, c->k_head}, {c->page_size, c->k_token}}},
           {c->v_pages, 2, c->head_dim, {{c->pages, c->v_page}, {c->kv_heads, c->v_head}, {c->page_size, c->v_token}}},
           {c->k_bounds, 2, c->k_bounds ? 2 * c->head_dim : 0, {{c->pages, c->b_page}, {c->kv_heads, c->b_head}}}} {}
  bool once() const {
    return of[0].once() && of[1].once() && of[2].once() && apart(of[0], of[1]) && apart(of[0], of[2]) && apart(of[1], of[2]);
  }
  bool apart_from(const Region& r) const { return apart(of[0], r) && apart(of[1], r) && apart(of[2], r); }
};

typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));

// Two binary32 values rounded to a 16-bit type, to nearest even.
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<f16_t>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){pin_f32(a), pin_f32(b)}, h2));
}
template <> __device__ __forceinline__ uint32_t pack_pair<bf16_t>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){a, b}, b2_t));
}

// Sum over the lanes up to this one.
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) {
#define TT_STEP(CTRL, ROWS) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
  TT_STEP(0x111, 0xF) TT_STEP(0x112, 0xF) TT_STEP(0x114, 0xF) TT_STEP(0x118, 0xF)     // within rows of 16
#undef TT_STEP
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);      // row 0's sum to row 1, row 2's to row 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);      // the first half's to the second
  return v;
}

// Which of the call's tokens are a row's: cu int32 [rows + 1], or `each` tokens for every row.  Values of cu
// outside 0 .. tokens count as the nearest inside, so that nothing lies outside the operands.
struct RowTokens {
  const int32_t* cu;
  int rows, tokens, each;
  __device__ __forceinline__ int begin(int r) const { return cu ? min(max(cu[r], 0), tokens) : r * each; }
  // (row, first token, tokens)
  __device__ __forceinline__ int count(int r, int* first) const {
    const int a = begin(r);
    *first = a;
    return max(0, begin(r + 1) - a);
  }
  // The last row whose first unit, begin / per + extra r, is at most x: units of `per` tokens (or a part of one)
  // are dealt to the rows in order, and a row of n tokens takes no more than n / per + extra of them.
  // Called by whole waves.
  __device__ __forceinline__ int find(int64_t x, int64_t num, int64_t per, int extra) const {
    int below = 0;
    const int lane = threadIdx.x & 63;
    for (int r0 = 0; r0 < rows; r0 += 64) {
      const int r = r0 + lane;
      const bool in = r < rows && (int64_t)begin(min(r, rows - 1)) * num / per + (int64_t)extra * r <= x;
      const int n = __popcll(__builtin_amdgcn_ballot_w64(in));
      below += n;
      if (n < 64) break;
    }
    return max(0, below - 1);
  }
};

// The row of one of the call's tokens (rows when it is behind the last one), its place in the row and the row's count:
// for single lanes, by halving.
__device__ __forceinline__ int row_of(const RowTokens& of, int token, int* place, int* count) {
  if (of.cu == nullptr) {
    const int r = token / of.each;
    *place = token - r * of.each;
    *count = of.each;
    return r;
  }
  int a = 0, b = of.rows;                // the last row that begins at or before the token
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (of.begin(mid) <= token) a = mid;
    else b = mid;
  }
  int first;
  *count = of.count(a, &first);
  *place = token - first;
  return *place >= 0 && *place < *count ? a : of.rows;
}

}  // namespace tt
