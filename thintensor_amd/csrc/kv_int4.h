// The 4-bit KV cache as the kernels see it, and the checks of its descriptor
// (layout: tt_int4_cache in thintensor_hip.h).
#pragma once

#include "tt_abi_internal.h"
#include "tt_regions.h"

namespace tt {

// What an entry point that takes a cache can check on the host.
inline int check_cache(const tt_int4_cache* c, int64_t rows, const char* what) {
  TT_REQUIRE(c != nullptr, "%s: null cache", what);
  TT_REQUIRE(c->k_codes && c->k_scales && c->v_codes && c->v_scales, "%s: null cache pointer", what);
  TT_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim must be 64, 128 or 256", what);
  TT_REQUIRE((c->group_size == 32 || c->group_size == 64 || c->group_size == 128) && c->group_size <= c->head_dim,
             "%s: group_size must be 32, 64 or 128 and at most head_dim", what);
  TT_REQUIRE(c->capacity > 0 && c->capacity % 32 == 0 && c->capacity < (1LL << 30),
             "%s: capacity must be a multiple of 32 tokens (below 2^30)", what);
  TT_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 65535 && c->batch > 0, "%s: bad batch / kv_heads", what);
  TT_REQUIRE(rows >= 0 && rows <= c->batch && rows <= 65535, "%s: %lld rows in a cache of %lld sequences (65535 at most)",
             what, (long long)rows, (long long)c->batch);
  // a lane of the attention reads the scale pairs of head_dim / 4 dims at once
  const int64_t pairs = c->head_dim / 4 > c->group_size ? 2 : 1;
  TT_REQUIRE(aligned(c->k_codes, 16) && aligned(c->v_codes, 16) && aligned(c->v_scales, 16),
             "%s: cache codes and v_scales must be 16-byte aligned", what);
  TT_REQUIRE(aligned(c->k_scales, 4 * (uintptr_t)pairs), "%s: cache k_scales must be %d-byte aligned", what, (int)(4 * pairs));
  TT_REQUIRE(c->kc_seq % 4 == 0 && c->kc_head % 4 == 0 && c->vc_seq % 4 == 0 && c->vc_head % 4 == 0 &&
                 c->vs_seq % 8 == 0 && c->vs_head % 8 == 0,
             "%s: cache strides must keep codes and v_scales of sequences and heads 16-byte aligned", what);
  TT_REQUIRE(c->ks_seq % (2 * pairs) == 0 && c->ks_head % (2 * pairs) == 0,
             "%s: cache strides must keep k_scales of sequences and heads %d-byte aligned", what, (int)(4 * pairs));
  return TT_OK;
}

// What sequences 0 .. rows - 1 of a cache take up: codes and scales of K, of V.
struct CacheRegions {
  Region of[4];
  CacheRegions(const tt_int4_cache* c, int64_t rows)
      : of{{c->k_codes, 4, c->capacity * c->head_dim / 8, {{rows, c->kc_seq}, {c->kv_heads, c->kc_head}}},
           {c->k_scales, 2, c->capacity * c->head_dim / c->group_size * 2, {{rows, c->ks_seq}, {c->kv_heads, c->ks_head}}},
           {c->v_codes, 4, c->capacity * c->head_dim / 8, {{rows, c->vc_seq}, {c->kv_heads, c->vc_head}}},
           {c->v_scales, 2, c->capacity * c->head_dim / c->group_size * 2, {{rows, c->vs_seq}, {c->kv_heads, c->vs_head}}}} {}
  // every byte of one sequence, head and array alone
  bool once() const {
    for (int i = 0; i < 4; i++) {
      if (!of[i].once()) return false;
      for (int j = 0; j < i; j++)
        if (!apart(of[i], of[j])) return false;
    }
    return true;
  }
  bool apart_from(const Region& r) const { return apart(of[0], r) && apart(of[1], r) && apart(of[2], r) && apart(of[3], r); }
};

}  // namespace tt
