// Appending to the paged cache with the rotation on the way (angles and rotation as in rotary.hip).
//
// What bounds it is memory: every value is read and written once.  One launch holds two kinds of workgroups.
// Those of keys and values take the tokens of one row that fall into one page, for some KV heads: a page's bounds
// then have one writer, which keeps the extremes of its places in registers and joins them in LDS, and no atomics
// are needed.  Those of queries take a few tokens with all their heads.
// 16384 tokens, 64 + 8 heads x 128, take 136 to 144 us (4.8 TB/s; a large copy 5.0), 517 and less of 12 rows with bounds, 40 +
// 10 heads, 15 to 17; one token of eight rows 4.8 (4.5 a call in a graph).  One workgroup for each head and page instead of
// several heads leaves short runs to the launch; one piece requested at a time 20.6 and 146 (loads wait behind stores).
// A page's tokens are not divided, so few heads and large pages leave CUs without work: 2048 tokens of one row, 16 + 2 heads
// x 256, take 63 us in pages of 256 tokens (18 workgroups) and 11 in pages of 16, 32 + 8 heads x 128 36 and 16.
#include "paged.h"
#include "tt_common.h"
#include "tt_eight.h"

#include <type_traits>

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
  int runs, head_groups, group_heads;      // workgroups of keys and values: runs x groups of KV heads
  int q_tokens;                            // tokens of a workgroup of queries
};

// The tokens of one row that fall into one page: tokens first + from .. of the call, slot slot0 of the page on.
struct Run {
  int64_t first, start, logical;           // the row's first token and its position; the page's place in the table
  int from, to;
  int32_t id;                              // the page, or -1
};
__device__ __forceinline__ Run run_of(const AppendParams& P, int x) {
  Run r;
  const int page = (int)P.c.page_size;
  int row, unit, first, n;
  if (P.of.cu && P.of.rows <= 64) {        // a row for each lane, what is known of it in one request
    const int lane = threadIdx.x & 63, mine = min(lane, P.of.rows - 1);
    int my_first;
    const int my_n = P.of.count(mine, &my_first), my_start = P.starts[mine];
    const int before = my_first / page + 2 * mine;
    row = max(0, __popcll(__builtin_amdgcn_ballot_w64(lane < P.of.rows && before <= x)) - 1);
    unit = x - __builtin_amdgcn_readlane(before, row);
    first = __builtin_amdgcn_readlane(my_first, row);
    n = __builtin_amdgcn_readlane(my_n, row);
    r.start = __builtin_amdgcn_readlane(my_start, row);
  } else {
    if (P.of.cu) {
      row = __builtin_amdgcn_readfirstlane(P.of.find(x, 1, page, 2));
      n = P.of.count(row, &first);
      unit = x - (first / page + 2 * row);
    } else {
      const int units = P.of.each / page + 2;
      row = x / units;
      unit = x - row * units;
      n = P.of.count(row, &first);
    }
    r.start = P.starts[row];
  }
  r.first = first;
  r.logical = (r.start >> __builtin_ctz(page)) + unit;      // floor, of negative positions too
  const int64_t a = r.logical * page - r.start, b = a + page;
  r.from = (int)(a > 0 ? (a < n ? a : n) : 0);
  r.to = (int)(b < n ? b : n);
  r.id = r.logical >= 0 && r.logical < P.table_pages ? P.table[row * P.table_row + r.logical] : -1;
  if (r.id >= P.c.pages || r.id < 0) r.id = -1;
  return r;
}

// cos and sin times the amplitude of `n` tokens' angles, to turn[token][half] and turn[token][half + ...].
template <typename F>
__device__ __forceinline__ void form_turns(const AppendParams& P, float* turn, int n, F&& position) {
  const int half = P.rotary >> 1;
  for (int v = threadIdx.x; v < n * half; v += 256) {
    const int tk = v / half, i = v - tk * half;
    const double t = (double)position(tk) * P.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * (float)(t - __builtin_rint(t)), &s, &c);
    turn[tk * P.rotary + i] = c * P.amplitude;
    turn[tk * P.rotary + half + i] = s * P.amplitude;
  }
}

// Eight binary32 values rounded to a 16-bit type by the conversion instruction.
template <typename T> __device__ __forceinline__ uint4 rounded(const float* v) {
  return make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]), pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7]));
}

template <typename T> constexpr uint32_t kInfinity = 0x7c00;
template <> constexpr uint32_t kInfinity<bf16_t> = 0x7f80;

// Two 16-bit floats as integers in their order (-0 below +0; NaN beyond the infinity of its sign), and back.
typedef short ss2_t __attribute__((ext_vector_type(2)));
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_keys(uint32_t w) {
  return w ^ (__builtin_bit_cast(uint32_t, __builtin_bit_cast(ss2_t, w) >> 15) | 0x80008000u);
}
__device__ __forceinline__ uint32_t from_keys(uint32_t k) {
  return k ^ (~__builtin_bit_cast(uint32_t, __builtin_bit_cast(ss2_t, k) >> 15) | 0x80008000u);
}
__device__ __forceinline__ uint32_t keys_min(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(us2_t, a), __builtin_bit_cast(us2_t, b)));
}
__device__ __forceinline__ uint32_t keys_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2_t, a), __builtin_bit_cast(us2_t, b)));
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A place of a head: eight pairs of the half layout (two pieces of eight dims), four of the interleaved one (one
// piece), or a piece to copy.
template <typename T, bool INTERLEAVED> struct Turned {
  static constexpr int NP = INTERLEAVED ? 1 : 2;
  Eight<T> a, b;
  __device__ __forceinline__ void load(const T* x, int d0, int d1, bool copy) {
    a.load(x + d0);
    if (NP == 2 && !copy) b.load(x + d1);
  }
  __device__ __forceinline__ void turn(const float* cs, int half, int u) {
    float ra[8], rb[8];
    if (INTERLEAVED) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float c = cs[4 * u + e], s = cs[half + 4 * u + e], x = a.get(2 * e), y = a.get(2 * e + 1);
        ra[2 * e] = x * c - y * s;
        ra[2 * e + 1] = y * c + x * s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float c = cs[8 * u + e], s = cs[half + 8 * u + e], x = a.get(e), y = b.get(e);
        ra[e] = x * c - y * s;
        rb[e] = y * c + x * s;
      }
      b.v = rounded<T>(rb);
    }
    a.v = rounded<T>(ra);
  }
  __device__ __forceinline__ void store(T* o, int d0, int d1, bool copy) const {
    if (NP == 2 && !copy) b.store(o + d1);
    a.store(o + d0);
  }
};

// f(0) .. f(N - 1), each with its own code: indexes of registers have to be known
template <int N, typename F> __device__ __forceinline__ void each_of(F&& f) {
  if constexpr (N > 0) {
    each_of<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

constexpr int kAhead = 4;                  // requested together, so that loads do not wait behind stores
constexpr int kTurnFloats = 4096;          // of LDS: tokens whose angles are formed at once, times rotary

// Rows whose vectors start on 16-byte boundaries and whose parts come in whole pieces of eight dims.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_vec_kernel(AppendParams P) {
  __shared__ __attribute__((aligned(16))) float turn_s[kTurnFloats];
  constexpr int NP = INTERLEAVED ? 1 : 2;
  const int dim = (int)P.c.head_dim, half = P.rotary >> 1, tid = threadIdx.x;
  const int turns = P.rotary / (8 * NP), units = turns + (dim - P.rotary) / 8;
  const int rows = 256 / units, r0 = tid / units, u = tid - r0 * units;
  const bool copy = u >= turns;
  const int d0 = copy ? P.rotary + 8 * (u - turns) : 8 * u, d1 = copy ? d0 : d0 + half;
  typedef Turned<T, INTERLEAVED> Piece;
  const int kv_groups = P.runs * P.head_groups;

  if ((int)blockIdx.x >= kv_groups) {
    // ---- queries
    const int t0 = ((int)blockIdx.x - kv_groups) * P.q_tokens, tokens = min(P.q_tokens, P.of.tokens - t0);
    const int total = r0 < rows ? tokens * P.heads : 0;
    Piece x[kAhead];
    auto at = [&](int r, int* tk, int* h) __attribute__((always_inline)) {
      *tk = r / P.heads;
      *h = r - *tk * P.heads;
    };
    auto load = [&](int r) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        int tk, h;
        at(min(r + k * rows, max(total - 1, 0)), &tk, &h);
        x[k].load(reinterpret_cast<const T*>(P.q) + (int64_t)(t0 + tk) * P.q_token + h * P.q_head, d0, d1, copy);
      }
    };
    load(r0);
    __shared__ int64_t pos_s[64];
    __shared__ int in_row[64];
    __shared__ int cu_s[257], start_s[256];
    const bool by_lds = P.of.cu && P.of.rows <= 256;
    if (by_lds) {                          // the rows' bounds and positions in one request, halved in LDS
      for (int i = tid; i <= P.of.rows; i += 256) cu_s[i] = P.of.begin(i);
      if (tid < P.of.rows) start_s[tid] = P.starts[tid];
      lds_barrier();
    }
    if (tid < tokens) {
      int place, count, start = 0;
      const int r = by_lds ? row_of(RowTokens{cu_s, P.of.rows, P.of.tokens, 0}, t0 + tid, &place, &count) : row_of(P.of, t0 + tid, &place, &count);
      if (r < P.of.rows) start = by_lds ? start_s[r] : P.starts[r];
      in_row[tid] = r < P.of.rows;
      pos_s[tid] = r < P.of.rows ? (int64_t)start + place : 0;
    }
    lds_barrier();
    form_turns(P, turn_s, tokens, [&](int tk) { return pos_s[tk]; });
    lds_barrier();
    for (int r = r0; r < total; r += kAhead * rows) {
      if (r != r0) load(r);
      each_of<kAhead>([&](auto index) __attribute__((always_inline)) {
        constexpr int k = index;
        if (r + k * rows >= total) return;
        int tk, h;
        at(r + k * rows, &tk, &h);
        if (!in_row[tk]) return;
        if (!copy) x[k].turn(turn_s + tk * P.rotary, half, u);
        x[k].store(reinterpret_cast<T*>(P.q_out) + (int64_t)(t0 + tk) * P.o_token + h * P.o_head, d0, d1, copy);
      });
    }
    return;
  }

  // ---- keys and values
  const Run run = run_of(P, blockIdx.x / P.head_groups);
  if (run.from >= run.to || run.id < 0) return;
  const int kvh0 = (blockIdx.x % P.head_groups) * P.group_heads, heads = min(P.group_heads, (int)P.c.kv_heads - kvh0);
  const int n = run.to - run.from, slot0 = (int)(run.start + run.from - run.logical * P.c.page_size);
  const int64_t token0 = run.first + run.from;
  const T* k = reinterpret_cast<const T*>(P.k) + token0 * P.k_token + kvh0 * P.k_head;
  const T* v = reinterpret_cast<const T*>(P.v) + token0 * P.v_token + kvh0 * P.v_head;
  T* kp = reinterpret_cast<T*>(P.c.k_pages) + (int64_t)run.id * P.c.k_page + kvh0 * P.c.k_head + (int64_t)slot0 * P.c.k_token;
  T* vp = reinterpret_cast<T*>(P.c.v_pages) + (int64_t)run.id * P.c.v_page + kvh0 * P.c.v_head + (int64_t)slot0 * P.c.v_token;

  // a thread keeps one place of one head and walks over the tokens
  const int lanes = rows / heads, tk0 = r0 / heads, head = r0 - tk0 * heads;
  const bool works = tk0 < lanes;
  uint32_t lo[4 * NP], hi[4 * NP];         // extremes of its places, as integers
#pragma unroll
  for (int e = 0; e < 4 * NP; e++) {
    lo[e] = 0xffffffffu;
    hi[e] = 0u;
  }
  // values: pieces of all tokens and heads, the first ones requested before the keys
  const int pieces = dim / 8, v_per = heads * pieces, v_total = n * v_per;
  typedef uint32_t v4_t __attribute__((ext_vector_type(4)));
  v4_t y[kAhead];
  auto load_v = [&](int i) __attribute__((always_inline)) {
    each_of<kAhead>([&](auto index) __attribute__((always_inline)) {
      constexpr int a = index;
      const int j = min(i + a * 256, v_total - 1), tk = j / v_per, r = j - tk * v_per, h = r / pieces;
      y[a] = *reinterpret_cast<const v4_t*>(v + (int64_t)tk * P.v_token + h * P.v_head + 8 * (r - h * pieces));
    });
  };
  auto store_v = [&](int i) __attribute__((always_inline)) {
    each_of<kAhead>([&](auto index) __attribute__((always_inline)) {
      constexpr int a = index;
      const int j = i + a * 256, tk = j / v_per, r = j - tk * v_per, h = r / pieces;
      if (j < v_total) *reinterpret_cast<v4_t*>(vp + (int64_t)tk * P.c.v_token + h * P.c.v_head + 8 * (r - h * pieces)) = y[a];
    });
  };
  load_v(tid);
  const int chunk = P.rotary > 0 ? min(n, kTurnFloats / P.rotary) : n;
  for (int c0 = 0; c0 < n; c0 += chunk) {
    const int end = min(c0 + chunk, n);
    Piece x[kAhead];
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kAhead; i++)
        x[i].load(k + (int64_t)min(t + i * lanes, end - 1) * P.k_token + head * P.k_head, d0, d1, copy);
    };
    if (works) load(c0 + tk0);
    if (c0 > 0) lds_barrier();
    form_turns(P, turn_s, end - c0, [&](int tk) { return run.start + run.from + c0 + tk; });
    lds_barrier();
    if (works)
      for (int t = c0 + tk0; t < end; t += kAhead * lanes) {
        if (t != c0 + tk0) load(t);
        each_of<kAhead>([&](auto index) __attribute__((always_inline)) {
          constexpr int i = index;
          const int tt = t + i * lanes;
          if (tt >= end) return;
          if (!copy) x[i].turn(turn_s + (tt - c0) * P.rotary, half, u);
          x[i].store(kp + (int64_t)tt * P.c.k_token + head * P.c.k_head, d0, d1, copy);
          if (P.c.k_bounds) {
#pragma unroll
            for (int e = 0; e < 4 * NP; e++) {                // of the keys as they are stored
              if (e >= 4 && copy) break;
              const uint32_t k = to_keys(word_of(e < 4 ? x[i].a.v : x[i].b.v, e & 3));
              lo[e] = keys_min(lo[e], k);
              hi[e] = keys_max(hi[e], k);
            }
          }
        });
      }
  }
  store_v(tid);
  for (int i = tid + kAhead * 256; i < v_total; i += kAhead * 256) {
    load_v(i);
    store_v(i);
  }
  if (P.c.k_bounds == nullptr) return;
  // ---- a dim's extremes over the token lanes, where the angles were
  T* bp = reinterpret_cast<T*>(P.c.k_bounds) + (int64_t)run.id * P.c.b_page + kvh0 * P.c.b_head;
  const bool anew = slot0 == 0;
  const int words = heads * dim / 2;                         // (of all lanes no more than half of kTurnFloats)
  uint32_t* const lo_s = reinterpret_cast<uint32_t*>(turn_s);
  uint32_t* const hi_s = lo_s + kTurnFloats / 2;
  lds_barrier();
  if (works)
#pragma unroll
    for (int e = 0; e < 4 * NP; e++) {
      if (e >= 4 && copy) break;
      const int at = tk0 * words + (head * dim + (e < 4 ? d0 : d1)) / 2 + (e & 3);
      lo_s[at] = lo[e];
      hi_s[at] = hi[e];
    }
  lds_barrier();
  for (int i = tid; i < words; i += 256) {
    const int h = 2 * i / dim, d = 2 * i - h * dim;
    uint32_t* const b = reinterpret_cast<uint32_t*>(bp + h * P.c.b_head + d);
    uint32_t l = 0xffffffffu, m = 0u, old_l = 0, old_m = 0;
    if (!anew) {
      old_l = b[0];
      old_m = b[dim / 2];
    }
    for (int t = 0; t < lanes; t++) {
      l = keys_min(l, lo_s[t * words + i]);
      m = keys_max(m, hi_s[t * words + i]);
    }
    const uint32_t new_l = from_keys(l), new_m = from_keys(m);
    if (!anew) {
      l = keys_min(l, to_keys(old_l));
      m = keys_max(m, to_keys(old_m));
    }
    l = from_keys(l);
    m = from_keys(m);
#pragma unroll
    for (int s = 0; s < 32; s += 16) {     // a NaN stays: of the page's own extreme, of a key in both
      const uint32_t part = 0xffffu << s;
      auto nan = [&](uint32_t w) __attribute__((always_inline)) { return ((w >> s) & 0x7fffu) > kInfinity<T>; };
      const bool both = nan(new_l) || nan(new_m);
      const uint32_t quiet = 0x7fffu << s;
      if (both || nan(old_l)) l = (l & ~part) | quiet;
      if (both || nan(old_m)) m = (m & ~part) | quiet;
    }
    b[0] = l;
    b[dim / 2] = m;
  }
}

// Any strides, alignment and rotary dims: a thread per pair or copied dim, one token after another, all heads of a row's
// page by one workgroup.  (16384 tokens, 64 + 8 heads x 128, with q, or k and v, an element off a 16-byte boundary: 944 us instead
// of 129; 512, 32 + 8 heads, 327 instead of 11.)
template <typename T>
__global__ __launch_bounds__(256) void append_kernel(AppendParams P) {
  __shared__ float2 turn[128];
  const int dim = (int)P.c.head_dim, kvh = (int)P.c.kv_heads, half = P.rotary >> 1;
  const Run run = run_of(P, blockIdx.x);
  const bool place = run.id >= 0;
  const int slot0 = (int)(run.start + run.from - run.logical * P.c.page_size);
  T* kp = reinterpret_cast<T*>(P.c.k_pages) + (int64_t)run.id * P.c.k_page;
  T* vp = reinterpret_cast<T*>(P.c.v_pages) + (int64_t)run.id * P.c.v_page;
  for (int i = run.from; i < run.to; i++) {
    const int64_t token = run.first + i, pos = run.start + i;
    const int slot = slot0 + i - run.from;
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
  if (!place || P.c.k_bounds == nullptr || run.from >= run.to) return;
  __syncthreads();
  T* bp = reinterpret_cast<T*>(P.c.k_bounds) + (int64_t)run.id * P.c.b_page;
  for (int u = threadIdx.x; u < kvh * dim; u += 256) {
    const int h = u / dim, d = u - h * dim;
    T* b = bp + h * P.c.b_head + d;
    const T* x = kp + h * P.c.k_head + d;
    float lo = to_f32(slot0 == 0 ? x[0] : b[0]), hi = to_f32(slot0 == 0 ? x[0] : b[dim]);
    for (int s = slot0; s < slot0 + run.to - run.from; s++) {
      const float y = to_f32(x[s * P.c.k_token]);
      lo = __builtin_elementwise_minimum(lo, y);
      hi = __builtin_elementwise_maximum(hi, y);
    }
    store<T>(b, lo);
    store<T>(b + dim, hi);
  }
}

template <typename T>
static int launch_append(AppendParams& P, int64_t rows, int64_t tokens, hipStream_t st, const char* what) {
  const int64_t page = P.c.page_size, kvh = P.c.kv_heads;
  P.runs = (int)(P.of.cu ? tokens / page + 2 * rows : rows * (P.of.each / page + 2));
  bool vec = P.rotary % (P.interleaved ? 8 : 16) == 0 && aligned(P.k, 16) && aligned(P.v, 16) &&
             ((P.k_token | P.k_head | P.v_token | P.v_head) & 7) == 0;
  if (P.heads > 0) vec = vec && aligned(P.q, 16) && aligned(P.q_out, 16) && ((P.q_token | P.q_head | P.o_token | P.o_head) & 7) == 0;
  if (!vec) {
    hipLaunchKernelGGL((append_kernel<T>), dim3((unsigned)P.runs), dim3(256), 0, st, P);
    return check_launch(what);
  }
  const int64_t units = (P.interleaved ? P.rotary / 8 : P.rotary / 16) + (P.c.head_dim - P.rotary) / 8, in_flight = 256 / units;
  // KV heads of a workgroup: as many as have places among its threads, fewer where runs are long and few
  int64_t heads = kvh < in_flight ? kvh : in_flight;
  while (heads > 1 && tokens >= 8 * rows && P.runs * ((kvh + heads - 1) / heads) < 4 * device_cus()) heads = (heads + 1) / 2;
  P.group_heads = (int)heads;
  P.head_groups = (int)((kvh + heads - 1) / heads);
  // tokens of a workgroup of queries: kAhead places for each thread
  int64_t q_tokens = 1;
  if (P.heads > 0) {
    q_tokens = kAhead * in_flight / P.heads;
    if (tokens / (q_tokens > 0 ? q_tokens : 1) < 2 * device_cus()) q_tokens = 1;
    const int64_t most = P.rotary > 0 && kTurnFloats / P.rotary < 64 ? kTurnFloats / P.rotary : 64;
    q_tokens = q_tokens < 1 ? 1 : q_tokens > most ? most : q_tokens;
  }
  P.q_tokens = (int)q_tokens;
  const int64_t blocks = (int64_t)P.runs * P.head_groups + (P.heads > 0 ? (tokens + q_tokens - 1) / q_tokens : 0);
  TT_REQUIRE(blocks < (1 << 24), "%s: too many tokens and heads for one call", what);
  if (P.interleaved) hipLaunchKernelGGL((append_vec_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, P);
  else hipLaunchKernelGGL((append_vec_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, P);
  return check_launch(what);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == TT_F16 ? launch_append<f16_t>(P, rows, tokens, st, what) : launch_append<bf16_t>(P, rows, tokens, st, what);
}
