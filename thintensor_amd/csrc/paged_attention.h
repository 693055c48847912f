// Attention over the paged cache: what its kernels share.
//
// There are two jobs: the rows' own pages (every row's queries against the tokens that the row does not
// share), and the shared pages (all rows' queries against them, from row 0's table).  A launch of the kernel for many
// columns serves one, that for few may serve both.  Either way the queries of a KV head are columns: column c is
// query head c % per_kv of the job's token c / per_kv, sees the tokens lo <= t < hi, and a tile of keys meets
// all columns of a workgroup at once.
#pragma once

#include "paged.h"
#include "tt_common.h"

namespace tt {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16v_t __attribute__((ext_vector_type(16)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));

// Weights are 2^7 exp(s - m), where m follows the running maximum only when that is more than 2^8 past it: they
// stay below 2^15, and the smallest step of fp16 is 2^-31 of the largest.
constexpr float kPScale = 7.0f;
constexpr float kSlack = 8.0f;
constexpr int kMostParts = 1024;       // parts of a query that the join takes

// One job of a launch for few columns: workgroups in all and for a row (of 16 columns times the kernel's blocks each), the
// rows, tiles of a workgroup, the first of the parts that they leave.
struct FewJob {
  int blocks, row_tiles, rows, share, part0;
};

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
  int q_vec, out_vec;                                // vectors of q start on 16-byte boundaries, of out on 8-byte ones
  float scale_log2;                                  // scale * log2(e)
  const void* sinks;
  int sink_dtype;
  void* out;
  int64_t out_token, out_head;
  // what parts of a query's tokens leave: weighted sums [tokens, heads, parts, D], (maximum, sum) of their weights
  float* part_o;
  float2* part_ml;
  int parts;
  int shared_entries;                                // of the table: read from row 0's
  // a launch for few columns: the rows' own pages [0], the shared pages [1]; or for many, of one of them
  FewJob few[2];
  int wide;
  int shared_job, part0, share, row_tiles, tiles, ordered;
};

template <typename T> struct Bits16;
template <> struct Bits16<f16_t> {
  static constexpr uint32_t kExp = 0x7c00;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_pair<f16_t>(a, b); }
  static __device__ __forceinline__ float add_pair(uint32_t w, float c) {      // c + both halves
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), (h2){(_Float16)1.0f, (_Float16)1.0f}, c, false);
  }
  static __device__ __forceinline__ f4_t mfma16(u4_t a, u4_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v_t mfma32(u4_t a, u4_t b, f16v_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  }
};
template <> struct Bits16<bf16_t> {
  static constexpr uint32_t kExp = 0x7f80;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_pair<bf16_t>(a, b); }
  static __device__ __forceinline__ float add_pair(uint32_t w, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2_t, w), (b2_t){(__bf16)1.0f, (__bf16)1.0f}, c, false);
  }
  static __device__ __forceinline__ f4_t mfma16(u4_t a, u4_t b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v_t mfma32(u4_t a, u4_t b, f16v_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  }
};

__device__ __forceinline__ float sink_log2(const PagedParams& P, int h) {
  const float v = P.sink_dtype == TT_F32    ? reinterpret_cast<const float*>(P.sinks)[h]
                  : P.sink_dtype == TT_BF16 ? to_f32(reinterpret_cast<const bf16_t*>(P.sinks)[h])
                                            : to_f32(reinterpret_cast<const f16_t*>(P.sinks)[h]);
  return v * 0x1.715476p+0f;
}

template <typename T> __device__ __forceinline__ void store_four(T* p, f4_t v, int vec) {
  const u2_t w = {Bits16<T>::pack(v[0], v[1]), Bits16<T>::pack(v[2], v[3])};
  if (vec) {
    *reinterpret_cast<u2_t*>(p) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) p[e].bits = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  }
}

// What a query head's sums become: o scale[0], where m is the maximum that o and l carry.  A query that saw
// nothing has no weight and is 0.
__device__ __forceinline__ float finish_scale(const PagedParams& P, int h, float m, float l) {
  if (l == 0.0f) return 0.0f;
  if (P.sinks) {
    const float sk = sink_log2(P, h), top = fmaxf(m, sk), e = __builtin_amdgcn_exp2f(m - top);
    return e / (l * e + __builtin_amdgcn_exp2f(sk - top + kPScale));
  }
  return 1.0f / l;
}

// What column c of a job sees: [lo, hi).
struct Seen {
  int lo, hi;
};
__device__ __forceinline__ Seen seen_of(const PagedParams& P, bool shared_job, int n, int place, int count) {
  Seen s;
  s.hi = n - (count - 1 - place);
  s.lo = P.window > 0 ? max(0, s.hi - P.window) : 0;
  if (shared_job) s.hi = min(s.hi, P.shared);
  else s.lo = max(s.lo, P.shared);
  return s;
}
__device__ __forceinline__ int row_length(const PagedParams& P, int row) { return min(max(P.lengths[row], 0), P.max_length); }

// The pages of a row, or of a selection of them: entry e of the table (of the selection) in lane e - base, of 64 and
// the 64 after them, so that looking one up is a move between registers.  (Scalar loads of the table would be waited for
// with every read of LDS.)
struct PageLanes {
  const int32_t* table;
  const int32_t* shared_table;   // of the first `shared` entries
  const int32_t* sel;
  int shared, pages, count, valid;       // entries; of the table, of the selection; of the cache
  int base, id[2], logical[2];
  __device__ __forceinline__ void load(int slot, int from) {
    const int e = from + (int)(threadIdx.x & 63);
    if (sel) {
      const int l = sel[min(e, count - 1)];
      const bool ok = e < count && l >= 0 && l < pages;
      logical[slot] = ok ? l : -1;
      id[slot] = table[ok ? l : 0];
    } else {
      id[slot] = (e < shared ? shared_table : table)[min(e, pages - 1)];
    }
  }
  __device__ __forceinline__ void start(int entry) {
    base = entry;
    load(0, base);
    load(1, base + 64);
  }
  __device__ __forceinline__ void reach(int entry) {         // entries from this one on (at most 127 past base)
    if (entry - base >= 64) {
      base += 64;
      id[0] = id[1];
      logical[0] = logical[1];
      load(1, base + 64);
    }
  }
  __device__ __forceinline__ int pick(const int (&v)[2], int entry) const {
    const int at = entry - base;
    return at < 64 ? __builtin_amdgcn_readlane(v[0], at) : __builtin_amdgcn_readlane(v[1], at - 64);
  }
};

// Sixteen tokens of a KV head that begin at a multiple of sixteen: one page holds them.
struct Place {
  const char *k, *v;
  int t;             // their first token; past every length where there is none
  bool bad;          // no page
};
__device__ __forceinline__ Place place_of(const PagedParams& P, const PageLanes& L, const char* k, const char* v, int u) {
  Place p;
  const int entry = u >> P.page_shift, slot = u & ((1 << P.page_shift) - 1);
  const int logical = L.sel ? L.pick(L.logical, entry) : entry;
  const int32_t id = L.pick(L.id, entry);
  p.bad = (uint32_t)id >= (uint32_t)L.valid;
  const int64_t page = p.bad ? 0 : id;
  p.t = (uint32_t)logical >= (uint32_t)L.pages ? 0x7fffff00 : (logical << P.page_shift) + slot;
  p.k = k + 2 * (page * P.c.k_page + slot * P.c.k_token);
  p.v = v + 2 * (page * P.c.v_page + slot * P.c.v_token);
  return p;
}

// Orders this wave's LDS accesses for its other lanes: a wave's LDS operations execute in order, the
// compiler has to keep them so.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Four rows of sixteen 16-bit values in LDS, transposed: of each sixteen lanes, lane 4 r + x gives the address of
// row r's values 4 x ..  and lane i gets value i of the four rows.
__device__ __forceinline__ u2_t lds_transposed(const char* p) {
  typedef __attribute__((address_space(3))) s4_t* Lds;
  return __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p));
}

template <typename T> __device__ __forceinline__ bool any_not_finite(u4_t v) {
  bool r = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t e = v[i] & (0x10001u * Bits16<T>::kExp);
    r |= (e & 0xffffu) == Bits16<T>::kExp || (e >> 16) == Bits16<T>::kExp;
  }
  return r;
}

// Values of tokens that some columns of a tile see and others do not: a weight of 0 would turn an infinite or NaN
// value into NaN for those that do not see it.  Such values are taken out of the tile, and what they make of the columns
// that see them is noted in LDS, two bits for each column and dim: 1 infinity, 2 minus infinity, 3 NaN.  So is, for
// all dims, that a column sees a token which lies in no page.
struct Marks {
  uint32_t* bits;                // [columns][words]: sixteen dims a word
  const Seen* see;               // [columns]
  int columns, words;
  __device__ __forceinline__ void no_page(int t, int tokens) const {      // of tokens t .. t + tokens - 1
#pragma unroll 1
    for (int c = 0; c < columns; c++) {
      const Seen s = see[c];
      if (s.lo < t + tokens && s.hi > t && s.hi > s.lo)
#pragma unroll 1
        for (int w = 0; w < words; w++) atomicOr(&bits[c * words + w], 0xffffffffu);
    }
  }
  // eight values of token t from dim d on, in LDS
  template <typename T> __device__ __forceinline__ void take_odd(uint16_t* v, int t, int d) const {
    using B = Bits16<T>;
#pragma unroll 1
    for (int e = 0; e < 8; e++) {
      const uint32_t x = v[e];
      if ((x & B::kExp) != B::kExp) continue;
      v[e] = 0;
      const uint32_t kind = (x & 0x7fffu) != B::kExp ? 3u : x >> 15 ? 2u : 1u;
#pragma unroll 1
      for (int c = 0; c < columns; c++) {
        const Seen s = see[c];
        if (t >= s.lo && t < s.hi) atomicOr(&bits[c * words + (d + e) / 16], kind << (2 * ((d + e) % 16)));
      }
    }
  }
  __device__ __forceinline__ float marked(float o, int c, int d) const {
    const uint32_t kind = (bits[c * words + d / 16] >> (2 * (d % 16))) & 3u;
    const float inf = __builtin_bit_cast(float, 0x7f800000u);
    return kind == 0 ? o : kind == 1 ? o + inf : kind == 2 ? o - inf : __builtin_bit_cast(float, 0x7fc00000u);
  }
};

// paged_few.hip: blocks of up to few_columns() columns of a row and KV head; paged_many.hip: 128 or 256
constexpr int few_columns(int64_t head_dim) { return head_dim == 64 ? 64 : head_dim == 128 ? 32 : 16; }
int launch_paged_few(const PagedParams& P, int blocks16, hipStream_t st, const char* what);
int launch_paged_many(const PagedParams& P, int waves, int splits, hipStream_t st, const char* what);
inline int many_tile_tokens(int64_t head_dim) { return head_dim == 256 ? 32 : 64; }

}  // namespace tt
