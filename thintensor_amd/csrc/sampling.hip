// One token per row of logits from given uniform numbers: temperature, top-k, top-p, min-p
// (tt_sample_rows in thintensor_hip.h).
//
// Every cut keeps a beginning of one order (logit descending, index ascending), and the token is
// where the cumulative weight passes a target in the same order.  So nothing needs the whole order:
// a histogram over z = (max - x) / temperature says which bins the cuts and the target can fall into,
// and only the candidates in those bins are put in order.
//   1. every chunk of a row: largest and smallest logit;
//   2. every chunk: weight (and, for top-k, count) of each bin;
//   3. every chunk: the bins that the row's cuts can fall into, and their candidates;
//   4. one workgroup per row: candidates sorted, cuts and target resolved among them.
// Weights are exp(-z) in units of 2^-43, 64-bit integers: sums have no order, and a total is exact to
// 2^-43 of the largest weight per token, far below what tells two cumulative sums apart.
//
// Four launches: one row of 128256 fp16 logits takes 16.5 us (2.7, 5.1, 5.6 and 4.1 for the steps: a launch and
// one round trip to memory are 3 of each), 64 rows of 152064 in binary32 49 us (7.9, 16.2, 16.3, 9.8): every
// pass over the 39 MB takes 8 us at the 5 TB/s that the memory gives, the weights 8 us of vector instructions
// beside it, the third step its round trips before the candidates are known, the last one sorts.
//
// A row that leaves more than kMostCandidates candidates is searched digit by digit by its one workgroup,
// up to three searches of 0.17 ms each (128256 equal logits).  It takes thousands of logits in a border's bin:
// 10^6 of nearly equal weight, or equal ones, which 16-bit logits far from zero have as a rule -- from 16 to 32
// bf16 values lie 0.125 apart.  Rows of 201088 bf16 logits of standard deviation 2, temperature 1 to 2, top-p
// 0.9 or 0.95: around 0 one takes 21 to 34 us a call, 64 take 71; around 20 or -20 0.37 to 0.51 ms and 0.58 to 0.71.
#include "tt_abi_internal.h"
#include "tt_common.h"

namespace tt {

constexpr int kBins = 2048;             // the last one: what lies past kReach
// z that the bins reach to at most: further ones weigh 2^-44.7, less than half a unit.  (Four rows of 200000, half
// of them masked by -65504: 48 us, 0.8 ms with bins to 64, which leave more candidates than are sorted.)
constexpr double kReach = 31.0;
constexpr double kUnit = 8796093022208.0;   // 2^43
constexpr int kThreads = 256;           // of a chunk's workgroup
constexpr int kStep = 8 * kThreads;     // logits that it takes at a time
// of step 2, where fewer workgroups leave fewer bins to add (one row of 128256, 8 of 201088, 64 of 152064:
// 256 threads 17.0, 22.7 and 50.9 us a call, 512 16.5, 22.3 and 49.2, 1024 17.2, 21.7 and 50.1)
constexpr int kBinThreads = 512;
constexpr int kMostChunks = 256;
constexpr int kMostCandidates = 4096;   // that the last step sorts in LDS
constexpr int kFinalThreads = 1024;
constexpr int kCuts = 4;                // intervals of bins: top-k, top-p, min-p, the target

// What step 3 leaves for step 4: disjoint intervals of bins in increasing order (n of them, behind them
// empty ones), the weight and count before each and up to its end; whether top-k divides a bin.
struct alignas(16) SamplePlan {
  int n;
  int lo[kCuts], hi[kCuts];
  uint64_t before[kCuts], upto[kCuts];
  uint32_t rank_before[kCuts], rank_upto[kCuts];
  int k_cut;                            // whether top-k divides a bin
  uint32_t k;
  uint64_t k_mass;                      // otherwise: the weight that it keeps
  uint64_t total, m_before;             // all weight; the weight before min-p's interval
};

struct alignas(16) SampleRow {                      // scratch of one row
  uint64_t mass[kBins];
  uint32_t count[kBins];
  float2 range[kMostChunks];            // largest, smallest finite
  SamplePlan plan;
  uint32_t candidates;
  uint32_t pad[3];
  uint64_t list[kMostCandidates];
};
static_assert(sizeof(SampleRow) % 16 == 0, "rows keep their alignment");

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int vocab, vec;                       // vec: rows start on 16-byte boundaries
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  SampleRow* rows;
  int chunks, chunk;                    // chunks of a row and their logits, a multiple of kStep
  int bin_chunks, bin_chunk;            // those of step 2
  int64_t* tokens;
  float* probs;
};

// Order-preserving key of a logit above -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x + 0.0f;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kNegInf = 0xff800000u;
__device__ __forceinline__ bool live(float x) { return x > __builtin_bit_cast(float, kNegInf); }

// e^-z for z >= 0 in binary64, as p 2^n: z log2 e = -n + f, p = e^(f ln 2) by its Taylor polynomial
// (|f ln 2| <= 0.3466: the first term left out is below 2^-52 of it).
__device__ __forceinline__ double exp_neg(double z, int* n) {
  const double y = z * -1.4426950408889634074;
  const double r = __builtin_rint(y);
  const double g = __builtin_fma(r, -0.69314718055994530942, -z);
  const double g2 = __builtin_fma(r, -2.3190468138462996e-17, g);   // the rest of ln 2
  double p = 2.08767569878681e-09;                                   // 1/12!
  p = __builtin_fma(p, g2, 2.505210838544172e-08);
  p = __builtin_fma(p, g2, 2.755731922398589e-07);
  p = __builtin_fma(p, g2, 2.7557319223985893e-06);
  p = __builtin_fma(p, g2, 2.48015873015873e-05);
  p = __builtin_fma(p, g2, 0.0001984126984126984);
  p = __builtin_fma(p, g2, 0.001388888888888889);
  p = __builtin_fma(p, g2, 0.008333333333333333);
  p = __builtin_fma(p, g2, 0.041666666666666664);
  p = __builtin_fma(p, g2, 0.16666666666666666);
  p = __builtin_fma(p, g2, 0.5);
  p = __builtin_fma(p, g2, 1.0);
  p = __builtin_fma(p, g2, 1.0);
  *n = (int)r;
  return p;
}

// What a row's settings and range make of a logit.  A greedy row, and one whose largest logit is
// infinite, is `hard`: only the largest ones weigh.  Elsewhere -inf becomes an infinite z and NaN a NaN,
// which weigh nothing.
struct RowScale {
  double top, inv_t, y_per_x, bins_per_z;
  bool greedy, hard;
  __device__ RowScale(float2 range, float t) {
    greedy = !(t > 0.0f);
    hard = greedy || range.x == __builtin_bit_cast(float, 0x7f800000u);
    top = (double)range.x;
    inv_t = greedy ? 0.0 : 1.0 / (double)t;
    y_per_x = inv_t * -1.4426950408889634074;
    const double far = hard ? kReach : soft_z(range.y);
    // all of the range in bins 0 .. kBins - 2, or what lies below kReach of it
    const double most = far < kReach ? far : kReach;
    bins_per_z = most > 0.0 ? (kBins - 2) / most : 0.0;
  }
  __device__ double soft_z(float x) const { return (top - (double)x) * inv_t; }
  __device__ double z_of(float x) const {
    if (hard) return (double)x == top ? 0.0 : __builtin_inf();
    return soft_z(x);
  }
  __device__ int bin_of(double z) const { return (int)__builtin_fmin(z * bins_per_z, (double)(kBins - 1)); }
  __device__ double weight_of(double z) const {
    if (!(z < 700.0)) return 0.0;
    int n;
    const double p = exp_neg(z, &n);
    return __builtin_amdgcn_ldexp(p, n);
  }
  // In units: 2^w, w = 43 - z log2 e, as 2^n p(f) with n the nearest integer and p of degree ten through 1
  // at f = 0 and at Chebyshev points of -1/2 .. 1/2 (within 2^-50.6 of 2^f); w is off by less than 2^-45: three
  // roundings of 2^-53 in y_per_x times up to 44.7, and its own of 2^-48 (200000 random ones: 2^-46.7 at most).
  // Before it is rounded a weight is off by less than a thirtieth of a unit.  2^52 added leaves the rounded
  // integer in the low bits.  What weighs nothing, NaN included, ends as 2^-21.
  __device__ uint64_t soft_mass(float x) const {
    const double w = __builtin_fmax(__builtin_fma(top - (double)x, y_per_x, 43.0), -21.0);
    const double n = __builtin_rint(w), f = w - n;
    double p = 7.070977866508139e-09;
    p = __builtin_fma(p, f, 1.0205905413765595e-07);
    p = __builtin_fma(p, f, 1.3215451623221434e-06);
    p = __builtin_fma(p, f, 1.5252672924850737e-05);
    p = __builtin_fma(p, f, 0.00015403530424776529);
    p = __builtin_fma(p, f, 0.0013333558200794592);
    p = __builtin_fma(p, f, 0.009618129107618665);
    p = __builtin_fma(p, f, 0.05550410866465167);
    p = __builtin_fma(p, f, 0.24022650695910075);
    p = __builtin_fma(p, f, 0.6931471805599462);
    p = __builtin_fma(p, f, 1.0);
    const double v = __builtin_amdgcn_ldexp(p, (int)n) + 4503599627370496.0;
    return __builtin_bit_cast(uint64_t, v) - 0x4330000000000000ull;
  }
  __device__ uint64_t mass_of(float x) const {
    if (hard) return (double)x == top ? (uint64_t)kUnit : 0;
    return soft_mass(x);
  }
};

// A row's settings as they are given: requested together at a kernel's start (one that is not given is read
// from the uniform numbers, and not used).
struct RowSettings {
  float t, p, min_p, u;
  int32_t k;
  __device__ RowSettings(const SampleParams& P, int row) {
    const float a = (P.temperature ? P.temperature : P.uniforms)[row], b = (P.top_p ? P.top_p : P.uniforms)[row];
    const float c = (P.min_p ? P.min_p : P.uniforms)[row];
    const int32_t d = (P.top_k ? P.top_k : reinterpret_cast<const int32_t*>(P.uniforms))[row];
    u = P.uniforms[row];
    t = P.temperature ? a : 1.0f;
    p = P.top_p ? b : 1.0f;
    min_p = P.min_p ? c : 0.0f;
    k = P.top_k ? d : 0;
  }
  // top-k where it cuts the order (a greedy row keeps the first), else 0
  __device__ uint32_t top_k(bool greedy, int vocab) const {
    const int32_t n = greedy ? 1 : k;
    return n > 0 && n < vocab ? (uint32_t)n : 0u;
  }
};

template <typename T>
__device__ __forceinline__ float logit(const SampleParams& P, int row, int i) {
  return to_f32(reinterpret_cast<const T*>(P.logits)[row * P.row_stride + i]);
}

// Eight logits from i on, -inf past the vocabulary.
template <typename T>
__device__ __forceinline__ void logits8(const SampleParams& P, int row, int i, float x[8]) {
  const T* p = reinterpret_cast<const T*>(P.logits) + row * P.row_stride + i;
  if (P.vec && i + 8 <= P.vocab) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = piece_f32<T>(v, e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = i + e < P.vocab ? to_f32(p[e]) : __builtin_bit_cast(float, kNegInf);
  }
}

__device__ __forceinline__ float2 wave_range(float hi, float lo) {
#define TT_LEVEL(M) hi = fmaxf(hi, xor_partner<M>(hi)); lo = fminf(lo, xor_partner<M>(lo));
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
  return make_float2(hi, lo);
}

// The row's range from its chunks', by every wave, all lanes: requested first of what a kernel reads, since
// loads arrive in order.
struct RowRange {
  float2 v[kMostChunks / 64];
  __device__ RowRange(const SampleParams& P, int row) {
    const float2* r = P.rows[row].range;
    const float inf = __builtin_bit_cast(float, 0x7f800000u);
#pragma unroll
    for (int k = 0; k < kMostChunks / 64; k++) {
      const int c = (threadIdx.x & 63) + 64 * k;
      v[k] = c < P.chunks ? r[c] : make_float2(-inf, inf);
    }
  }
  __device__ float2 get() const {
    float2 w = v[0];
#pragma unroll
    for (int k = 1; k < kMostChunks / 64; k++) w = make_float2(fmaxf(w.x, v[k].x), fminf(w.y, v[k].y));
    return wave_range(w.x, w.y);
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_range_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  for (int b = c * kThreads + threadIdx.x; b < kBins; b += kThreads * P.chunks) {
    R.mass[b] = 0;
    R.count[b] = 0;
  }
  if (c == 0 && threadIdx.x == 0) R.candidates = 0;
  const float inf = __builtin_bit_cast(float, 0x7f800000u);
  float hi = -inf, lo = inf;
  const int end = min(P.vocab, (c + 1) * P.chunk);
#pragma unroll 2
  for (int i = c * P.chunk + 8 * (int)threadIdx.x; i < end; i += kStep) {
    float x[8];
    logits8<T>(P, row, i, x);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      hi = fmaxf(hi, x[e]);
      lo = fminf(lo, live(x[e]) ? x[e] : inf);
    }
  }
  __shared__ float2 ws[kThreads / 64];
  const float2 w = wave_range(hi, lo);
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    R.range[c] = make_float2(fmaxf(fmaxf(ws[0].x, ws[1].x), fmaxf(ws[2].x, ws[3].x)),
                             fminf(fminf(ws[0].y, ws[1].y), fminf(ws[2].y, ws[3].y)));
  }
}

template <typename T>
__global__ __launch_bounds__(kBinThreads) void sample_bins_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  __shared__ __attribute__((aligned(16))) uint64_t mass[kBins];
  __shared__ __attribute__((aligned(16))) uint32_t count[kBins];
  const int end = min(P.vocab, (c + 1) * P.bin_chunk);
  int i = c * P.bin_chunk + 8 * (int)threadIdx.x;
  const RowRange chunks(P, row);
  float x[8];
  if (i < end) logits8<T>(P, row, i, x);
  const RowSettings G(P, row);
  for (int b = threadIdx.x; b < kBins / 2; b += kBinThreads) {
    reinterpret_cast<ulonglong2*>(mass)[b] = make_ulonglong2(0, 0);
    reinterpret_cast<uint2*>(count)[b] = make_uint2(0, 0);
  }
  const RowScale S(chunks.get(), G.t);
  const bool counts = G.top_k(S.greedy, P.vocab) != 0;
  uint32_t far = 0;                     // of the last bin
  __syncthreads();
  while (i < end) {
    int b[8];
    uint64_t m[8];
    if (S.hard) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool is_top = (double)x[e] == S.top;
        b[e] = is_top ? 0 : kBins - 1;
        m[e] = is_top ? (uint64_t)kUnit : 0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        b[e] = S.bin_of(S.soft_z(x[e]));
        m[e] = S.soft_mass(x[e]);
      }
    }
    if (counts) {
#pragma unroll
      for (int e = 0; e < 8; e++) far += b[e] == kBins - 1 && live(x[e]);
    }
    const int next = i + 8 * kBinThreads;
    if (next < end) logits8<T>(P, row, next, x);
    // (what is not live lies in the last bin)
    if (counts) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (b[e] == kBins - 1) continue;
        atomicAdd(&count[b[e]], 1u);
        atomicAdd((unsigned long long*)&mass[b[e]], (unsigned long long)m[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (m[e]) atomicAdd((unsigned long long*)&mass[b[e]], (unsigned long long)m[e]);
      }
    }
    i = next;
  }
  if (counts && far) atomicAdd(&count[kBins - 1], far);
  __syncthreads();
  for (int k = threadIdx.x; k < kBins; k += kBinThreads) {
    if (mass[k]) atomicAdd((unsigned long long*)&R.mass[k], (unsigned long long)mass[k]);
    if (counts && count[k]) atomicAdd(&R.count[k], count[k]);
  }
}

// Sum over this lane and the ones before it in the wave: within rows of sixteen lanes, then over the rows.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define TT_LEVEL(CTRL, ROWS) v += dpp0<CTRL, ROWS>(v);
  TT_LEVEL(0x111, 0xf) TT_LEVEL(0x112, 0xf) TT_LEVEL(0x114, 0xf) TT_LEVEL(0x118, 0xf)   // row_shr 1, 2, 4, 8
  TT_LEVEL(0x142, 0xa) TT_LEVEL(0x143, 0xc)                                             // row_bcast 15, 31
#undef TT_LEVEL
  return v;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
#define TT_LEVEL(CTRL, ROWS) v += ((uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | dpp0<CTRL, ROWS>((uint32_t)v);
  TT_LEVEL(0x111, 0xf) TT_LEVEL(0x112, 0xf) TT_LEVEL(0x114, 0xf) TT_LEVEL(0x118, 0xf)
  TT_LEVEL(0x142, 0xa) TT_LEVEL(0x143, 0xc)
#undef TT_LEVEL
  return v;
}

// A row's cumulative histogram in LDS, where every wave searches it by itself: a look at the ends of its 64
// blocks of 32 bins, then one at a block, each a comparison in all lanes.  Blocks lie four banks apart.
struct CumBins {
  uint64_t m[kBins + 2 * (kBins / 32)];
  uint32_t n[kBins + 4 * (kBins / 32)];
  uint64_t wave_m[kThreads / 64];
  uint32_t wave_n[kThreads / 64];
  static __device__ __forceinline__ int at_m(int bin) { return bin + 2 * (bin >> 5); }
  static __device__ __forceinline__ int at_n(int bin) { return bin + 4 * (bin >> 5); }
  // weight and count of the bins up to this one
  __device__ uint64_t mass(int bin) const { return bin < 0 ? 0 : m[at_m(bin)]; }
  __device__ uint32_t count(int bin) const { return bin < 0 ? 0 : n[at_n(bin)]; }
  // The first bin with which the weight (count) reaches `want`; the last one if none does.
  __device__ int find_count(uint32_t want) const {
    const int lane = threadIdx.x & 63;
    const int block = __builtin_popcountll(__builtin_amdgcn_ballot_w64(n[at_n(32 * lane + 31)] < want));
    if (block == kBins / 32) return kBins - 1;
    return 32 * block + __builtin_popcount((uint32_t)__builtin_amdgcn_ballot_w64(n[at_n(32 * block + (lane & 31))] < want));
  }
  __device__ int find_mass(uint64_t want) const {
    const int lane = threadIdx.x & 63;
    const int block = __builtin_popcountll(__builtin_amdgcn_ballot_w64(m[at_m(32 * lane + 31)] < want));
    if (block == kBins / 32) return kBins - 1;
    return 32 * block + __builtin_popcount((uint32_t)__builtin_amdgcn_ballot_w64(m[at_m(32 * block + (lane & 31))] < want));
  }
};
static_assert(kBins == 64 * 32, "two looks of a wave");

// Eight bins of the histogram per thread.
struct BinPart {
  static constexpr int PER = kBins / kThreads;
  static_assert(PER == 8 && kThreads % 64 == 0, "a thread's bins lie in one block");
  uint64_t m[PER];
  uint32_t n[PER];
  __device__ void load(const SampleRow& R) {
    const ulonglong2* rm = reinterpret_cast<const ulonglong2*>(R.mass + threadIdx.x * PER);
    const uint4* rn = reinterpret_cast<const uint4*>(R.count + threadIdx.x * PER);
#pragma unroll
    for (int k = 0; k < PER / 2; k++) {
      const ulonglong2 v = rm[k];
      m[2 * k] = v.x; m[2 * k + 1] = v.y;
    }
#pragma unroll
    for (int k = 0; k < PER / 4; k++) {
      const uint4 v = rn[k];
      n[4 * k] = v.x; n[4 * k + 1] = v.y; n[4 * k + 2] = v.z; n[4 * k + 3] = v.w;
    }
  }
  __device__ void sum(CumBins& C) {     // two barriers
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
#pragma unroll
    for (int k = 1; k < PER; k++) {
      m[k] += m[k - 1];
      n[k] += n[k - 1];
    }
    const uint64_t mi = wave_scan(m[PER - 1]);
    const uint32_t ni = wave_scan(n[PER - 1]);
    if ((t & 63) == 63) {
      C.wave_m[wave] = mi;
      C.wave_n[wave] = ni;
    }
    __syncthreads();
    uint64_t mb = mi - m[PER - 1];
    uint32_t nb = ni - n[PER - 1];
#pragma unroll
    for (int w = 0; w < kThreads / 64 - 1; w++)
      if (w < wave) {
        mb += C.wave_m[w];
        nb += C.wave_n[w];
      }
    ulonglong2* pm = reinterpret_cast<ulonglong2*>(&C.m[CumBins::at_m(t * PER)]);
    uint4* pn = reinterpret_cast<uint4*>(&C.n[CumBins::at_n(t * PER)]);
#pragma unroll
    for (int k = 0; k < PER / 2; k++) pm[k] = make_ulonglong2(mb + m[2 * k], mb + m[2 * k + 1]);
#pragma unroll
    for (int k = 0; k < PER / 4; k++) pn[k] = make_uint4(nb + n[4 * k], nb + n[4 * k + 1], nb + n[4 * k + 2], nb + n[4 * k + 3]);
    __syncthreads();
  }
};

// What the cuts take from a row's settings.
struct Cuts {
  uint32_t k;                           // 0: none
  double p, min_p, u;
  bool use_p, use_m;
  __device__ Cuts(const RowSettings& G, bool greedy, int vocab) {
    k = G.top_k(greedy, vocab);
    u = G.u > 0.0f ? (G.u < 1.0f ? (double)G.u : 1.0 - 0x1p-24) : 0.0;
    use_p = G.p < 1.0f;
    p = G.p > 0.0f ? (double)G.p : 0.0;
    use_m = G.min_p > 0.0f;
    min_p = (double)G.min_p;
  }
  // The bins that min-p's last logit can lie in: around -log(min_p), which its rounding and that of a weight
  // move by less than 2^-48 of it and of 1 -- many bins where the temperature is high.
  __device__ void min_p_bins(const RowScale& S, int* lo, int* hi) const {
    const double z = S.greedy || !(min_p < 1.0) ? 0.0 : -log(min_p);
    const double room = __builtin_fma(z, 0x1p-48, 0x1p-48);
    *lo = __builtin_amdgcn_readfirstlane(S.bin_of(__builtin_fmax(z - room, 0.0)));
    *hi = __builtin_amdgcn_readfirstlane(S.bin_of(z + room));
  }
  // The cumulative weight that the last of top-p's share reaches first, and the one that the token does:
  // integers, so that every step compares alike.  Both are at most `mass` (p and u are 1 - 2^-24 at most).
  __device__ uint64_t reach(uint64_t mass) const {
    const double t = p * (double)mass;
    return t > 1.0 ? (uint64_t)__builtin_ceil(t) : 1;
  }
  __device__ uint64_t target(uint64_t mass) const { return (uint64_t)(u * (double)mass) + 1; }
};

// Steps of a chunk on their way at a time (64 rows of 152064: two 16.5 us, three 16.9, four 17.6).
constexpr int kDeep = 2;

template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_gather_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  // the histogram, then the chunk's candidates
  __shared__ __attribute__((aligned(16))) union {
    CumBins bins;
    uint64_t found[kMostCandidates];
  } U;
  __shared__ uint32_t n_found, base;
  const int end = min(P.vocab, (c + 1) * P.chunk);
  int i = c * P.chunk + 8 * (int)threadIdx.x;
  const RowRange chunks(P, row);
  BinPart part;
  part.load(R);
  float x[kDeep][8];
#pragma unroll
  for (int k = 0; k < kDeep; k++)
    if (i + k * kStep < end) logits8<T>(P, row, i + k * kStep, x[k]);
  const RowSettings G(P, row);
  const float2 range = chunks.get();
  if (!live(range.x)) return;
  if (threadIdx.x == 0) n_found = 0;
  part.sum(U.bins);
  const CumBins& B = U.bins;
  const RowScale S(range, G.t);
  const Cuts C(G, S.greedy, P.vocab);
  const uint64_t total = B.mass(kBins - 1);

  // ---- top-k: the bin of its last one; whole bins and the last bin (no weight) need no resolving
  uint64_t k_lo = total, k_hi = total;
  int k_bin = -1;
  if (C.k && C.k < B.count(kBins - 1)) {
    const int b = B.find_count(C.k);
    k_lo = k_hi = B.mass(b);
    if (B.count(b) != C.k && b != kBins - 1) {
      k_bin = b;
      k_lo = B.mass(b - 1);
    }
  }
  // ---- top-p and min-p, as far as the weight of top-k is known
  uint64_t kept_lo = k_lo, kept_hi = k_hi, m_before = 0;
  int p_lo = -1, p_hi = -2, m_lo = -1, m_hi = -2;
  if (C.use_p) {
    p_lo = B.find_mass(C.reach(k_lo));
    p_hi = k_bin < 0 ? p_lo : B.find_mass(C.reach(k_hi));
    if (p_lo < kBins - 1) kept_lo = min(kept_lo, B.mass(p_lo - 1));
    if (p_hi < kBins - 1) kept_hi = min(kept_hi, B.mass(p_hi));
  }
  if (C.use_m) {
    C.min_p_bins(S, &m_lo, &m_hi);
    m_before = B.mass(m_lo - 1);
    kept_lo = min(kept_lo, m_before);
    kept_hi = min(kept_hi, B.mass(m_hi));
  }
  // ---- the target, and disjoint intervals in order
  int lo[kCuts] = {k_bin < 0 ? kBins : k_bin, p_hi < p_lo ? kBins : p_lo, m_hi < m_lo ? kBins : m_lo, B.find_mass(C.target(kept_lo))};
  int hi[kCuts] = {k_bin, p_hi, m_hi, B.find_mass(C.target(kept_hi))};
#pragma unroll
  for (int a = 0; a < kCuts; a++) {
    hi[a] = min(hi[a], kBins - 2);      // the last bin weighs nothing
    if (hi[a] < lo[a]) lo[a] = kBins;
  }
#pragma unroll
  for (int a = 0; a < kCuts - 1; a++)
#pragma unroll
    for (int b = 0; b < kCuts - 1 - a; b++)
      if (lo[b + 1] < lo[b]) {
        const int l = lo[b], h = hi[b];
        lo[b] = lo[b + 1]; hi[b] = hi[b + 1];
        lo[b + 1] = l; hi[b + 1] = h;
      }
#pragma unroll
  for (int a = 1; a < kCuts; a++)
    if (lo[a] < kBins) {
      // joined with the one before where they touch; that one takes this place
      const bool touch = lo[a - 1] < kBins && lo[a] <= hi[a - 1] + 1;
      if (touch) {
        lo[a] = lo[a - 1];
        hi[a] = max(hi[a], hi[a - 1]);
        lo[a - 1] = kBins;
      }
    }
  if (c == 0 && threadIdx.x < kCuts) {  // the plan, for the last step: an interval per lane, empty ones last
    SamplePlan& L = R.plan;
    const int a = (int)threadIdx.x;
    const int l = a == 0 ? lo[0] : a == 1 ? lo[1] : a == 2 ? lo[2] : lo[3];
    const int h = a == 0 ? hi[0] : a == 1 ? hi[1] : a == 2 ? hi[2] : hi[3];
    const bool used = l < kBins;
    const uint32_t all = (uint32_t)__builtin_amdgcn_ballot_w64(used), below = (1u << a) - 1;
    const int n = __builtin_popcount(all);
    const int at = used ? __builtin_popcount(all & below) : n + __builtin_popcount(~all & below);
    L.lo[at] = l;
    L.hi[at] = used ? h : -1;
    L.before[at] = used ? B.mass(l - 1) : 0;
    L.upto[at] = used ? B.mass(h) : 0;
    L.rank_before[at] = used ? B.count(l - 1) : 0;
    L.rank_upto[at] = used ? B.count(h) : 0;
    if (a == 0) {
      L.n = n;
      L.k_cut = k_bin >= 0;
      L.k = C.k;
      L.k_mass = k_hi;
      L.total = total;
      L.m_before = m_before;
    }
  }
  __syncthreads();                      // the histogram is not read any more
  // ---- this chunk's candidates
  int first = kBins;                    // most logits are past every interval
  int last = -1;
#pragma unroll
  for (int a = 0; a < kCuts; a++)
    if (lo[a] < kBins) {
      first = min(first, lo[a]);
      last = max(last, hi[a]);
    }
  // logits outside [x_lo, x_hi] cannot be in them: the borders in z, with room for their rounding
  float x_lo = __builtin_bit_cast(float, 0xff7fffffu), x_hi = __builtin_bit_cast(float, 0x7f800000u);
  if (!S.hard && S.bins_per_z > 0.0) {
    const double t = 1.0 / (S.bins_per_z * S.inv_t), lo_v = S.top - (last + 1) * t, hi_v = S.top - first * t;
    const double room = 0x1p-20 * (__builtin_fabs(S.top) + (last + 1) * t);
    x_lo = fmaxf(x_lo, (float)(lo_v - room));
    x_hi = (float)(hi_v + room);
  }
  for (; i < end; i += kDeep * kStep) {
#pragma unroll
    for (int k = 0; k < kDeep; k++) {
      const int at = i + k * kStep;
      if (at >= end) break;
      uint32_t maybe = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) maybe |= x[k][e] >= x_lo && x[k][e] <= x_hi ? 1u << e : 0u;
      if (maybe) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if (!((maybe >> e) & 1u)) continue;
          const int b = S.bin_of(S.z_of(x[k][e]));
          if (b < first || b > last) continue;
          bool in = false;
#pragma unroll
          for (int a = 0; a < kCuts; a++) in |= b >= lo[a] && b <= hi[a];
          if (!in) continue;
          // past the list's end the row is searched another way
          const uint32_t j = atomicAdd(&n_found, 1u);
          if (j < (uint32_t)kMostCandidates) U.found[j] = ((uint64_t)key_of(x[k][e]) << 32) | (uint32_t)~(uint32_t)(at + e);
        }
      }
      if (at + kDeep * kStep < end) logits8<T>(P, row, at + kDeep * kStep, x[k]);
    }
  }
  __syncthreads();
  const uint32_t n = n_found;
  if (n == 0) return;
  if (threadIdx.x == 0) base = atomicAdd(&R.candidates, n);
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < n; j += kThreads)
    if (base + j < (uint32_t)kMostCandidates) R.list[base + j] = U.found[j];
}

// Value of lane ^ M of a 64-bit integer.
template <int M>
__device__ __forceinline__ uint64_t xor64(uint64_t v) {
  const uint32_t hi = __builtin_bit_cast(uint32_t, xor_partner<M>(__builtin_bit_cast(float, (uint32_t)(v >> 32))));
  const uint32_t lo = __builtin_bit_cast(uint32_t, xor_partner<M>(__builtin_bit_cast(float, (uint32_t)v)));
  return ((uint64_t)hi << 32) | lo;
}

// Sorts n keys, one per thread, largest first: n is a power of two, 64 to 1024, and the threads past it have
// left.  Bitonic: partners within a wave by lane exchange, others in LDS, where two halves of `buf` take turns.
__device__ uint64_t sort_one(uint64_t v, int n, uint64_t* half) {
  const int t = threadIdx.x;
  uint64_t* buf = half;
  auto keep = [&](uint64_t mine, uint64_t other, int j, int k) {
    const bool larger = ((t & j) == 0) == ((t & k) == 0);   // this thread keeps the larger one
    return (mine < other) == larger ? other : mine;
  };
  auto within = [&](int k, int from) {
    if (from >= 32) v = keep(v, xor64<32>(v), 32, k);
    if (from >= 16) v = keep(v, xor64<16>(v), 16, k);
    if (from >= 8) v = keep(v, xor64<8>(v), 8, k);
    if (from >= 4) v = keep(v, xor64<4>(v), 4, k);
    if (from >= 2) v = keep(v, xor64<2>(v), 2, k);
    v = keep(v, xor64<1>(v), 1, k);
  };
  for (int k = 2; k <= 64; k <<= 1) within(k, k >> 1);
  for (int k = 128; k <= n; k <<= 1) {
    for (int j = k >> 1; j >= 64; j >>= 1) {
      buf[t] = v;
      lds_barrier();
      v = keep(v, buf[t ^ j], j, k);
      buf = buf == half ? half + kFinalThreads : half;
    }
    within(k, 32);
  }
  return v;
}

// More keys: four per thread, n a power of two, 2048 at least, and the threads past it only meet the barriers.
// Runs of k keys descend where key index & k is 0.
struct SortKeys {
  uint64_t v[4];
  // a pair within the thread: the first keeps the larger one where `down`
  __device__ __forceinline__ void pair(int i, int j, bool down) {
    const uint64_t x = v[i], y = v[j];
    const bool swap = (x < y) == down;
    v[i] = swap ? y : x;
    v[j] = swap ? x : y;
  }
  __device__ __forceinline__ void keep(int k, uint64_t other, bool larger) { v[k] = (v[k] < other) == larger ? other : v[k]; }
  template <int M>
  __device__ __forceinline__ void lanes(bool down) {
#pragma unroll
    for (int k = 0; k < 4; k++) keep(k, xor64<M>(v[k]), !(threadIdx.x & M) == down);
  }
  __device__ void sort(int n, uint64_t* buf) {
    const int t = threadIdx.x;
    pair(0, 1, true);
    pair(2, 3, false);
    for (int k = 4; k <= n; k <<= 1) {
      const bool down = !(t & (k >> 2));
      for (int j = k >> 3; j >= 64; j >>= 1) {
        ulonglong2* mine = reinterpret_cast<ulonglong2*>(buf + 4 * t);
        mine[0] = make_ulonglong2(v[0], v[1]);
        mine[1] = make_ulonglong2(v[2], v[3]);
        __syncthreads();
        const ulonglong2* other = reinterpret_cast<const ulonglong2*>(buf + 4 * (t ^ j));
        const ulonglong2 a = other[0], b = other[1];
        __syncthreads();
        const bool larger = !(t & j) == down;
        keep(0, a.x, larger);
        keep(1, a.y, larger);
        keep(2, b.x, larger);
        keep(3, b.y, larger);
      }
      if (k >= 256) lanes<32>(down);
      if (k >= 128) lanes<16>(down);
      if (k >= 64) lanes<8>(down);
      if (k >= 32) lanes<4>(down);
      if (k >= 16) lanes<2>(down);
      if (k >= 8) lanes<1>(down);
      pair(0, 2, down);
      pair(1, 3, down);
      pair(0, 1, down);
      pair(2, 3, down);
    }
  }
};

struct Found {           // answer of a search
  uint64_t mass;         // cumulative weight up to and including the element
  uint64_t key;          // the element
};

// A candidate list that does not fit: the elements of one interval are searched by the digits of
// their keys and indexes, over the row itself: the element of rank `rank`, or without one (0) the first whose
// cumulative weight reaches `want`.  Digits that all elements
// share are found first and passed over; once a key is settled its elements weigh the same and are
// counted.  A thread adds up what falls to one digit in a row before it meets the others in LDS.
template <typename T>
__device__ Found search_digits(const SampleParams& P, int row, const RowScale& S, const SamplePlan& L, int a,
                               uint32_t rank, uint64_t want, uint64_t* dm, uint32_t* dn, uint64_t* answer) {
  const int lo = L.lo[a], hi = L.hi[a];
  auto each = [&](auto f) __attribute__((always_inline)) {   // (key with index, logit) of the interval's elements
    for (int i = 8 * (int)threadIdx.x; i < P.vocab; i += 8 * kFinalThreads) {
      float x[8];
      logits8<T>(P, row, i, x);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (!live(x[e])) continue;
        const int b = S.bin_of(S.z_of(x[e]));
        if (b >= lo && b <= hi) f(((uint64_t)key_of(x[e]) << 32) | (uint32_t)~(uint32_t)(i + e), x[e]);
      }
    }
  };
  uint64_t mass = L.before[a];
  uint32_t count = L.rank_before[a];
  if (threadIdx.x == 0) {
    answer[0] = ~0ull;
    answer[1] = 0;
  }
  __syncthreads();
  uint64_t all = ~0ull, any = 0;
  each([&](uint64_t key, float) {
    all &= key;
    any |= key;
  });
  atomicAnd((unsigned long long*)&answer[0], (unsigned long long)all);
  atomicOr((unsigned long long*)&answer[1], (unsigned long long)any);
  __syncthreads();
  const uint64_t same = ~(answer[0] ^ answer[1]);   // bits that every key has alike
  uint64_t prefix = answer[0] & same;               // of these, and of the digits found
  uint64_t unit = 0;                                // the weight of one element, where the key is settled
  for (int shift = 56; shift >= 0; shift -= 8) {
    const uint64_t above = shift == 56 ? 0 : ~0ull << (shift + 8);
    if (((same >> shift) & 255u) == 255u) continue;
    const bool counted = (same | above) >> 32 == 0xffffffffull;
    if (counted && unit == 0) unit = S.mass_of(of_key((uint32_t)(prefix >> 32)));
    __syncthreads();
    for (int b = threadIdx.x; b < 256; b += kFinalThreads) {
      dm[b] = 0;
      dn[b] = 0;
    }
    __syncthreads();
    int digit = -1;
    uint32_t n = 0;
    uint64_t m = 0;
    auto flush = [&]() __attribute__((always_inline)) {
      if (digit < 0) return;
      atomicAdd(&dn[digit], n);
      if (!counted) atomicAdd((unsigned long long*)&dm[digit], (unsigned long long)m);
    };
    each([&](uint64_t key, float x) {
      if (((key ^ prefix) & above) != 0) return;
      const int d = (int)(key >> shift) & 255;
      if (d != digit) {
        flush();
        digit = d;
        n = 0;
        m = 0;
      }
      n++;
      if (!counted) m += S.mass_of(x);
    });
    flush();
    __syncthreads();
    if (threadIdx.x == 0) {
      int pick = -1;
      uint64_t pm = mass;
      uint32_t pn = count;
      for (int b = 255; b >= 0; b--) {
        if (dn[b] == 0) continue;
        pick = b;
        pm = mass;
        pn = count;
        mass += counted ? dn[b] * unit : dm[b];
        count += dn[b];
        if (rank ? count >= rank : mass >= want) break;
      }
      answer[0] = pm;
      answer[1] = pn;
      answer[2] = (uint64_t)pick;
    }
    __syncthreads();
    mass = answer[0];
    count = (uint32_t)answer[1];
    prefix = (prefix & ~(255ull << shift)) | ((answer[2] & 255u) << shift);
  }
  mass += S.mass_of(of_key((uint32_t)(prefix >> 32)));   // the element itself
  __syncthreads();                                               // answer may be written again
  return Found{mass, prefix};
}

template <typename T>
__global__ __launch_bounds__(kFinalThreads) void sample_final_kernel(SampleParams P) {
  constexpr int PER = kMostCandidates / kFinalThreads, WAVES = kFinalThreads / 64;
  const int row = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  SampleRow& R = P.rows[row];
  static_assert(PER == 4, "keys of a thread");
  __shared__ __attribute__((aligned(16))) uint64_t list[kMostCandidates];
  __shared__ uint64_t digits[256];
  __shared__ __attribute__((aligned(16))) uint64_t wave_sum[WAVES];
  __shared__ uint64_t answer[4];
  __shared__ unsigned long long kept_m;
  const RowRange chunks(P, row);
  // the plan and the number of candidates, a word per lane
  constexpr int WORDS = sizeof(SamplePlan) / 4;
  static_assert(WORDS < 64 && offsetof(SampleRow, candidates) == offsetof(SampleRow, plan) + sizeof(SamplePlan), "one load of a wave");
  const uint32_t words = reinterpret_cast<const uint32_t*>(&R.plan)[min(t & 63, WORDS)];
  uint64_t mine = R.list[t];            // (used where the list is that long)
  const RowSettings G(P, row);
  const float2 range = chunks.get();
  if (!live(range.x)) {
    if (t == 0) {
      P.tokens[row] = -1;
      if (P.probs) P.probs[row] = 0.0f;
    }
    return;
  }
  const uint32_t n = __builtin_amdgcn_readlane(words, WORDS);
  SamplePlan L;
  {
    uint32_t w[WORDS];
#pragma unroll
    for (int k = 0; k < WORDS; k++) w[k] = __builtin_amdgcn_readlane(words, k);
    __builtin_memcpy(&L, w, sizeof(L));
  }
  const RowScale S(range, G.t);
  const Cuts C(G, S.greedy, P.vocab);
  if (t == 0) {
    kept_m = L.m_before;
    answer[1] = L.total;
  }
  uint64_t k_mass = L.k_mass, kept, key = 0;
  if (n <= (uint32_t)kMostCandidates) {
    // ---- the candidates in order: thread t holds entries t per .. t per + per - 1
    const bool one = n <= (uint32_t)kFinalThreads;
    const int per = one ? 1 : PER;
    int size = 64;
    while (size < (int)n) size <<= 1;
    if (one && 64 * wave >= size) return;   // (a barrier waits for the waves that are left)
    uint64_t entry[PER] = {};
    if (one) {
      if (t >= (int)n) mine = 0;
      entry[0] = sort_one(mine, size, list);
    } else {
      SortKeys keys;
      const ulonglong2* p = reinterpret_cast<const ulonglong2*>(R.list + PER * t);
      const ulonglong2 x = p[0], y = p[1];
      keys.v[0] = x.x; keys.v[1] = x.y; keys.v[2] = y.x; keys.v[3] = y.y;
#pragma unroll
      for (int k = 0; k < PER; k++) keys.v[k] = PER * t + k < (int)n ? keys.v[k] : 0;
      keys.sort(size, list);
#pragma unroll
      for (int k = 0; k < PER; k++) entry[k] = keys.v[k];
    }
    // ---- their cumulative weights and ranks: of the candidates, plus what lies between their intervals
    uint64_t w[PER], sum = 0;
    int bins[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      bins[k] = -1;
      w[k] = 0;
      if (k < per && t * per + k < (int)n) {
        const float x = of_key((uint32_t)(entry[k] >> 32));
        bins[k] = S.bin_of(S.z_of(x));
        w[k] = S.mass_of(x);
      }
      sum += w[k];
    }
    const uint64_t incl = wave_scan(sum);
    if ((t & 63) == 63) wave_sum[wave] = incl;
    __syncthreads();
    uint64_t before = incl - sum;
#pragma unroll
    for (int v = 0; v < WAVES - 1; v++) before += v < wave ? wave_sum[v] : 0;
    uint64_t gap[kCuts], inside = 0;
    uint32_t rank_gap[kCuts], rank_inside = 0;
#pragma unroll
    for (int a = 0; a < kCuts; a++) {
      gap[a] = L.before[a] - inside;
      rank_gap[a] = L.rank_before[a] - rank_inside;
      inside += L.upto[a] - L.before[a];
      rank_inside += L.rank_upto[a] - L.rank_before[a];
    }
    uint64_t full[PER];                 // weight up to and including an entry
    uint32_t rank[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      before += w[k];
      full[k] = before + gap[0];
      rank[k] = rank_gap[0];
#pragma unroll
      for (int a = 1; a < kCuts; a++)
        if (bins[k] >= L.lo[a]) {
          full[k] = before + gap[a];
          rank[k] = rank_gap[a];
        }
      rank[k] += (uint32_t)(t * per + k) + 1;
    }
    // the entry with which the weight reaches `want`
    auto reaches = [&](int k, uint64_t want) __attribute__((always_inline)) {
      return bins[k] >= 0 && full[k] >= want && full[k] - w[k] < want;
    };
    // ---- top-k
    if (L.k_cut) {
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (bins[k] >= 0 && rank[k] == L.k) answer[0] = full[k];
      __syncthreads();
      k_mass = answer[0];
    }
    kept = k_mass;
    // ---- top-p and min-p
    if (C.use_p) {
      const uint64_t want = C.reach(k_mass);
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (reaches(k, want)) answer[1] = full[k];
    }
    if (C.use_m) {
#pragma unroll
      for (int k = 0; k < PER; k++)
        if (bins[k] >= 0) {
          const double z = S.z_of(of_key((uint32_t)(entry[k] >> 32)));
          if (z == 0.0 || S.weight_of(z) >= C.min_p) atomicMax(&kept_m, (unsigned long long)full[k]);
        }
    }
    if (C.use_p || C.use_m) {
      __syncthreads();
      if (C.use_p) kept = min(kept, answer[1]);
      // a min_p above 1 keeps the first alone
      if (C.use_m) kept = min(kept, C.min_p > 1.0 ? (uint64_t)kUnit : (uint64_t)kept_m);
    }
    // ---- the token
    const uint64_t want = C.target(kept);
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (reaches(k, want)) answer[2] = entry[k];
    __syncthreads();
    key = answer[2];
  } else {
    const SamplePlan& Q = R.plan;       // (picked from by number)
    // the interval that an answer lies in
    auto holding = [&](uint64_t want) {
      int a = 0;
      while (a + 1 < Q.n && Q.upto[a] < want) a++;
      return a;
    };
    uint32_t* dn = reinterpret_cast<uint32_t*>(list);
    __syncthreads();
    if (L.k_cut) {
      int a = 0;
      while (a + 1 < Q.n && Q.rank_before[a + 1] < Q.k) a++;
      k_mass = search_digits<T>(P, row, S, Q, a, Q.k, 0, digits, dn, answer).mass;
    }
    kept = k_mass;
    if (C.use_p) {
      const uint64_t want = C.reach(k_mass);
      kept = min(kept, search_digits<T>(P, row, S, Q, holding(want), 0, want, digits, dn, answer).mass);
    }
    if (C.use_m) {
      // every logit from min-p's interval on that passes
      uint64_t some = 0;
      int m_lo, m_hi;
      C.min_p_bins(S, &m_lo, &m_hi);
      for (int i = t; i < P.vocab; i += kFinalThreads) {
        const float x = logit<T>(P, row, i);
        if (!live(x)) continue;
        const double z = S.z_of(x);
        const int bz = S.bin_of(z);
        if (bz >= m_lo && bz <= m_hi && (z == 0.0 || S.weight_of(z) >= C.min_p)) some += S.mass_of(x);
      }
      __syncthreads();
      if (some) atomicAdd(&kept_m, (unsigned long long)some);
      __syncthreads();
      kept = min(kept, C.min_p > 1.0 ? (uint64_t)kUnit : (uint64_t)kept_m);
    }
    const uint64_t want = C.target(kept);
    key = search_digits<T>(P, row, S, Q, holding(want), 0, want, digits, dn, answer).key;
  }
  if (t == 0) {
    P.tokens[row] = (int64_t)(uint32_t)~(uint32_t)key;
    if (P.probs) P.probs[row] = (float)(S.weight_of(S.z_of(of_key((uint32_t)(key >> 32)))) * kUnit / (double)kept);
  }
}

template <typename T>
static int launch_sample(const SampleParams& P, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)P.chunks, (unsigned)rows), block(kThreads);
  hipLaunchKernelGGL((sample_range_kernel<T>), grid, block, 0, st, P);
  int rc = check_launch("sample_rows");
  if (rc) return rc;
  hipLaunchKernelGGL((sample_bins_kernel<T>), dim3((unsigned)P.bin_chunks, (unsigned)rows), dim3(kBinThreads), 0, st, P);
  if ((rc = check_launch("sample_rows"))) return rc;
  hipLaunchKernelGGL((sample_gather_kernel<T>), grid, block, 0, st, P);
  if ((rc = check_launch("sample_rows"))) return rc;
  hipLaunchKernelGGL((sample_final_kernel<T>), dim3((unsigned)rows), dim3(kFinalThreads), 0, st, P);
  return check_launch("sample_rows");
}

}  // namespace tt

using namespace tt;

extern "C" int64_t tt_sample_rows_scratch_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || vocab <= 0) return TT_ERR_INVALID;
  return rows * (int64_t)sizeof(SampleRow);
}

extern "C" int tt_sample_rows(const void* logits, int64_t row_stride, int dtype, int64_t rows, int64_t vocab,
                              const float* uniforms, const float* temperature, const int32_t* top_k, const float* top_p,
                              const float* min_p, void* scratch, int64_t scratch_bytes, int64_t* tokens, float* probs,
                              void* stream) {
  const char* what = "sample_rows";
  // 2^20 weights of 2^43 units add up below 2^64
  TT_REQUIRE(rows >= 0 && rows <= 65535 && vocab > 0 && vocab <= (1 << 20), "%s: at most 65535 rows of 2^20 logits", what);
  TT_REQUIRE(valid_out_dtype(dtype), "%s: logits must be fp16, bf16 or fp32", what);
  if (rows == 0) return TT_OK;
  TT_REQUIRE(logits && uniforms && tokens && scratch, "%s: null pointer", what);
  TT_REQUIRE(aligned(scratch, 16) && scratch_bytes >= rows * (int64_t)sizeof(SampleRow), "%s: scratch too small", what);
  SampleParams P{};
  P.logits = logits; P.row_stride = row_stride; P.vocab = (int)vocab;
  P.vec = aligned(logits, 16) && row_stride % (dtype == TT_F32 ? 4 : 8) == 0;
  P.uniforms = uniforms; P.temperature = temperature; P.top_k = top_k; P.top_p = top_p; P.min_p = min_p;
  P.rows = reinterpret_cast<SampleRow*>(scratch);
  // chunks: a step of logits each while that leaves the chip four workgroups per CU (two larger ones)
  auto cut = [&](int64_t step, int64_t groups, int* chunks, int* chunk) {
    const int64_t steps = (vocab + step - 1) / step, most = (groups + rows - 1) / rows;
    const int64_t fit = most < kMostChunks ? most : kMostChunks, per = (steps + fit - 1) / fit;
    *chunk = (int)(per * step);
    *chunks = (int)((steps + per - 1) / per);
  };
  const int64_t cus = device_cus();
  cut(kStep, 4 * cus, &P.chunks, &P.chunk);
  cut(8 * kBinThreads, 2 * cus, &P.bin_chunks, &P.bin_chunk);
  P.tokens = tokens; P.probs = probs;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TT_F16) return launch_sample<f16_t>(P, rows, st);
  if (dtype == TT_BF16) return launch_sample<bf16_t>(P, rows, st);
  return launch_sample<float>(P, rows, st);
}
