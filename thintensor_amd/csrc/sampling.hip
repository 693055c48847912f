// One token per row of logits from given uniform numbers: temperature, top-k, top-p, min-p
// (tt_sample_rows in thintensor_hip.h).
//
// Every cut keeps a beginning of one order (logit descending, index ascending), and the token is
// where the cumulative weight passes a target in the same order.  So nothing needs the whole order:
// a histogram over z = (max - x) / temperature says which bins the cuts and the target can fall into,
// and only the candidates in those bins are put in order.
//   1. every chunk of a row: largest and smallest logit;
//   2. every chunk: count and weight of each bin;
//   3. every chunk: the candidates, gathered from the bins that the row's cuts can fall into;
//   4. one workgroup per row: candidates sorted, cuts and target resolved among them.
// Weights are exp(-z) in units of 2^-43, 64-bit integers: sums have no order, and a total is exact to
// 2^-43 of the largest weight per token, far below what tells two cumulative sums apart.
#include "tt_abi_internal.h"
#include "tt_common.h"

namespace tt {

constexpr int kBins = 2048;             // the last one: weights below 2^-43, which count as 0
constexpr double kReach = 64.0;         // z that the bins reach to at most
constexpr double kUnit = 8796093022208.0;   // 2^43
constexpr int kMostChunks = 64;
constexpr int kMostCandidates = 4096;   // that the last step sorts in LDS
constexpr int kFinalThreads = 1024;

struct SampleRow {                      // scratch of one row
  uint64_t mass[kBins];
  uint32_t count[kBins];
  float2 range[kMostChunks];            // largest, smallest finite
  uint32_t candidates;
  uint32_t pad[3];
  uint64_t list[kMostCandidates];
};

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  int64_t vocab;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  SampleRow* rows;
  int chunks, chunk;                    // chunks of a row and their elements
  int64_t* tokens;
  float* probs;
};

// Order-preserving key of a logit; NaN and -inf as 0 (never taken), -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x + 0.0f;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  if (!(x > __builtin_bit_cast(float, 0xff800000u))) return 0u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ bool live(float x) { return x > __builtin_bit_cast(float, 0xff800000u); }

// What a row's settings and range make of a logit.
struct RowScale {
  double top, inv_t, bins_per_z;
  bool greedy;
  __device__ RowScale(const SampleParams& P, int row, float largest, float smallest) {
    const float t = P.temperature ? P.temperature[row] : 1.0f;
    greedy = !(t > 0.0f);
    top = (double)largest;
    inv_t = greedy ? 0.0 : 1.0 / (double)t;
    const double far = greedy ? kReach : z_of(smallest);
    // all of the range in bins 0 .. kBins - 2, or what lies below kReach of it
    const double most = far < kReach ? far : kReach;
    bins_per_z = most > 0.0 ? (kBins - 2) / most : 0.0;
  }
  __device__ double z_of(float x) const {
    if ((double)x == top) return 0.0;
    if (greedy) return __builtin_inf();
    return (top - (double)x) * inv_t;
  }
  __device__ int bin_of(double z) const {
    const double b = z == 0.0 ? 0.0 : z * bins_per_z;
    return b < (double)(kBins - 1) ? (int)b : kBins - 1;
  }
  __device__ double weight_of(double z) const { return exp(-z); }
  __device__ uint64_t mass_of(double z) const { return (uint64_t)(weight_of(z) * kUnit + 0.5); }
};

template <typename T>
__device__ __forceinline__ float logit(const SampleParams& P, int row, int64_t i) {
  return to_f32(reinterpret_cast<const T*>(P.logits)[row * P.row_stride + i]);
}

__device__ __forceinline__ float2 row_range(const SampleParams& P, int row) {
  const float2* r = P.rows[row].range;
  float hi = __builtin_bit_cast(float, 0xff800000u), lo = __builtin_bit_cast(float, 0x7f800000u);
  for (int c = 0; c < P.chunks; c++) {
    hi = fmaxf(hi, r[c].x);
    lo = fminf(lo, r[c].y);
  }
  return make_float2(hi, lo);
}

template <typename T>
__global__ __launch_bounds__(256) void sample_range_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  for (int b = c * 256 + threadIdx.x; b < kBins; b += 256 * P.chunks) {
    R.mass[b] = 0;
    R.count[b] = 0;
  }
  if (c == 0 && threadIdx.x == 0) R.candidates = 0;
  const float inf = __builtin_bit_cast(float, 0x7f800000u);
  float hi = -inf, lo = inf;
  const int64_t end = min(P.vocab, (int64_t)(c + 1) * P.chunk);
  for (int64_t i = (int64_t)c * P.chunk + threadIdx.x; i < end; i += 256) {
    const float x = logit<T>(P, row, i);
    hi = fmaxf(hi, x);
    if (live(x)) lo = fminf(lo, x);
  }
  __shared__ float hs[4], ls[4];
#define TT_LEVEL(M) hi = fmaxf(hi, xor_partner<M>(hi)); lo = fminf(lo, xor_partner<M>(lo));
  TT_LEVEL(1) TT_LEVEL(2) TT_LEVEL(4) TT_LEVEL(8) TT_LEVEL(16) TT_LEVEL(32)
#undef TT_LEVEL
  if ((threadIdx.x & 63) == 0) {
    hs[threadIdx.x >> 6] = hi;
    ls[threadIdx.x >> 6] = lo;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    R.range[c] = make_float2(fmaxf(fmaxf(hs[0], hs[1]), fmaxf(hs[2], hs[3])),
                             fminf(fminf(ls[0], ls[1]), fminf(ls[2], ls[3])));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  for (int b = threadIdx.x; b < kBins; b += 256) {
    mass[b] = 0;
    count[b] = 0;
  }
  const float2 range = row_range(P, row);
  const RowScale S(P, row, range.x, range.y);
  __syncthreads();
  const int64_t end = min(P.vocab, (int64_t)(c + 1) * P.chunk);
  for (int64_t i = (int64_t)c * P.chunk + threadIdx.x; i < end; i += 256) {
    const float x = logit<T>(P, row, i);
    if (!live(x)) continue;
    const double z = S.z_of(x);
    const int b = S.bin_of(z);
    atomicAdd(&count[b], 1u);
    if (b < kBins - 1) atomicAdd((unsigned long long*)&mass[b], (unsigned long long)S.mass_of(z));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += 256)
    if (count[b]) {
      atomicAdd(&R.count[b], count[b]);
      atomicAdd((unsigned long long*)&R.mass[b], (unsigned long long)mass[b]);
    }
}

// The cumulative histogram of a row and the bins that its cuts and target can fall into.
struct Bins {
  uint64_t mass[kBins + 1];             // before each bin
  uint32_t count[kBins + 1];
  uint64_t wave_mass[kFinalThreads / 64];
  uint32_t wave_count[kFinalThreads / 64];
  int at;                               // answer of a search
};

// Fills B from the row's histogram; THREADS threads, kBins / THREADS bins each.
template <int THREADS>
__device__ void cumulate(const SampleRow& R, Bins& B) {
  constexpr int PER = kBins / THREADS;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint64_t m[PER], ms = 0;
  uint32_t n[PER], ns = 0;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    m[k] = ms;
    n[k] = ns;
    ms += R.mass[t * PER + k];
    ns += R.count[t * PER + k];
  }
  uint64_t mi = ms;
  uint32_t ni = ns;
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t mo = __shfl_up((unsigned long long)mi, d);
    const uint32_t no = __shfl_up(ni, d);
    if (lane >= d) {
      mi += mo;
      ni += no;
    }
  }
  if (lane == 63) {
    B.wave_mass[wave] = mi;
    B.wave_count[wave] = ni;
  }
  __syncthreads();
  uint64_t mb = mi - ms;
  uint32_t nb = ni - ns;
  for (int w = 0; w < wave; w++) {
    mb += B.wave_mass[w];
    nb += B.wave_count[w];
  }
#pragma unroll
  for (int k = 0; k < PER; k++) {
    B.mass[t * PER + k] = mb + m[k];
    B.count[t * PER + k] = nb + n[k];
  }
  if (t == THREADS - 1) {
    B.mass[kBins] = mb + ms;
    B.count[kBins] = nb + ns;
  }
  __syncthreads();
}

// First bin whose cumulative weight (the bin's own included) is at least / more than target;
// kBins - 1 if none is.  The same for every thread.
__device__ __forceinline__ int bin_at_least(const Bins& B, double target) {
  int lo = 0, hi = kBins - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((double)B.mass[mid + 1] >= target) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
__device__ __forceinline__ int bin_above(const Bins& B, double target) {
  int lo = 0, hi = kBins - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((double)B.mass[mid + 1] > target) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
__device__ __forceinline__ int bin_of_rank(const Bins& B, uint32_t rank) {   // rank 1 .. count
  int lo = 0, hi = kBins - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (B.count[mid + 1] >= rank) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// A row's cuts as intervals of bins; an interval is empty where nothing needs resolving.
struct Cuts {
  uint32_t k;                           // rank of the last kept by top-k; 0: no cut
  double p, min_p, u;
  bool use_p, use_m;
  int k_bin, p_lo, p_hi, m_lo, m_hi, u_lo, u_hi;
  uint64_t k_mass;                      // where k_bin < 0: the weight kept by top-k
  __device__ Cuts(const SampleParams& P, int row, const RowScale& S, const Bins& B) {
    const uint32_t total = B.count[kBins];
    const int32_t tk = S.greedy ? 1 : P.top_k ? P.top_k[row] : 0;
    const float tp = P.top_p ? P.top_p[row] : 1.0f, mp = P.min_p ? P.min_p[row] : 0.0f;
    const float un = P.uniforms[row];
    u = un > 0.0f ? (un < 1.0f ? (double)un : 1.0 - 0x1p-24) : 0.0;
    k = tk > 0 && (uint32_t)tk < total ? (uint32_t)tk : 0;
    use_p = tp < 1.0f;
    p = tp > 0.0f ? (double)tp : 0.0;
    use_m = mp > 0.0f;
    min_p = (double)mp;
    // top-k: a bin it divides has to be resolved; the last bin weighs nothing
    k_bin = -1;
    k_mass = B.mass[kBins];
    uint64_t lo = k_mass, hi = k_mass;
    if (k) {
      const int b = bin_of_rank(B, k);
      if (B.count[b + 1] == k || b == kBins - 1) {
        k_mass = lo = hi = B.mass[b + 1];
      } else {
        k_bin = b;
        lo = B.mass[b];
        hi = B.mass[b + 1];
      }
    }
    p_lo = p_hi = -1;
    uint64_t kept_lo = lo, kept_hi = hi;
    if (use_p) {
      p_lo = bin_at_least(B, p * (double)lo);
      p_hi = bin_at_least(B, p * (double)hi);
      kept_lo = min(kept_lo, B.mass[p_lo]);
      kept_hi = min(kept_hi, B.mass[p_hi + 1]);
    }
    m_lo = m_hi = -1;
    if (use_m) {
      const double z = min_p < 1.0 ? -log(min_p) : 0.0;
      const int b = S.greedy ? 0 : S.bin_of(z);
      m_lo = max(0, b - 1);
      m_hi = min(kBins - 1, b + 1);
      kept_lo = min(kept_lo, B.mass[m_lo]);
      kept_hi = min(kept_hi, B.mass[m_hi + 1]);
    }
    u_lo = bin_above(B, u * (double)kept_lo);
    u_hi = bin_above(B, u * (double)kept_hi);
  }
  __device__ bool needs(int b) const {
    return b < kBins - 1 && (b == k_bin || (b >= p_lo && b <= p_hi) || (b >= m_lo && b <= m_hi) || (b >= u_lo && b <= u_hi));
  }
};

template <typename T>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleParams P) {
  const int row = blockIdx.y, c = blockIdx.x;
  SampleRow& R = P.rows[row];
  __shared__ Bins B;
  __shared__ uint64_t found[1024];
  __shared__ uint32_t n_found, base;
  if (threadIdx.x == 0) n_found = 0;
  const float2 range = row_range(P, row);
  if (!live(range.x)) return;
  const RowScale S(P, row, range.x, range.y);
  cumulate<256>(R, B);
  const Cuts C(P, row, S, B);
  const int64_t end = min(P.vocab, (int64_t)(c + 1) * P.chunk);
  for (int64_t i0 = (int64_t)c * P.chunk; i0 < end; i0 += 1024) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int64_t i = i0 + 256 * k + threadIdx.x;
      const float x = i < end ? logit<T>(P, row, i) : __builtin_bit_cast(float, 0xff800000u);
      if (live(x) && C.needs(S.bin_of(S.z_of(x)))) {
        const uint32_t at = atomicAdd(&n_found, 1u);
        found[at] = ((uint64_t)key_of(x) << 32) | (uint32_t)~(uint32_t)i;
      }
    }
    __syncthreads();
    const uint32_t n = n_found;
    __syncthreads();                    // every thread has read it before it counts again
    if (n) {
      if (threadIdx.x == 0) {
        base = atomicAdd(&R.candidates, n);
        n_found = 0;
      }
      __syncthreads();
      for (uint32_t j = threadIdx.x; j < n; j += 256)
        if (base + j < (uint32_t)kMostCandidates) R.list[base + j] = found[j];
      __syncthreads();
    }
  }
}

// Sorts n (a power of two, at most kMostCandidates) keys in LDS, largest first.
__device__ void sort_descending(uint64_t* a, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kFinalThreads) {
        const int l = 2 * i - (i & (j - 1)), r = l + j;
        const uint64_t x = a[l], y = a[r];
        const bool desc = (l & k) == 0;
        if ((x < y) == desc) {
          a[l] = y;
          a[r] = x;
        }
      }
      __syncthreads();
    }
}

struct Found {           // answers of the last step's searches
  uint64_t mass;         // cumulative weight up to and including the element
  uint64_t key;          // the element
};

// A candidate list that does not fit: the elements of bins lo .. hi are searched by the digits of
// their keys and indexes, over the row itself.  mode 0: the element of rank `rank`; 1: the first
// whose cumulative weight is at least target; 2: the first whose is more.
template <typename T>
__device__ Found search_digits(const SampleParams& P, int row, const RowScale& S, const Bins& B, int lo, int hi, int mode,
                               uint32_t rank, double target, uint64_t* dm, uint32_t* dn, uint64_t* answer) {
  uint64_t prefix = 0, mass = B.mass[lo];
  uint32_t count = B.count[lo];
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += kFinalThreads) {
      dm[b] = 0;
      dn[b] = 0;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < P.vocab; i += kFinalThreads) {
      const float x = logit<T>(P, row, i);
      if (!live(x)) continue;
      const double z = S.z_of(x);
      const int b = S.bin_of(z);
      const uint64_t key = ((uint64_t)key_of(x) << 32) | (uint32_t)~(uint32_t)i;
      if (b < lo || b > hi || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
      const int digit = (int)(key >> shift) & 255;
      atomicAdd(&dn[digit], 1u);
      atomicAdd((unsigned long long*)&dm[digit], (unsigned long long)S.mass_of(z));
    }
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
        mass += dm[b];
        count += dn[b];
        if (mode == 0 ? count >= rank : mode == 1 ? (double)mass >= target : (double)mass > target) break;
      }
      answer[0] = pm;
      answer[1] = ((uint64_t)pn << 32) | (uint32_t)pick;
      answer[2] = dm[pick < 0 ? 0 : pick];
    }
    __syncthreads();
    mass = answer[0];
    count = (uint32_t)(answer[1] >> 32);
    prefix = (prefix << 8) | (uint32_t)(answer[1] & 255u);
    if (shift == 0) mass += answer[2];
    __syncthreads();
  }
  return Found{mass, prefix};
}

template <typename T>
__global__ __launch_bounds__(kFinalThreads) void sample_final_kernel(SampleParams P) {
  const int row = blockIdx.x, t = threadIdx.x;
  SampleRow& R = P.rows[row];
  __shared__ Bins B;
  __shared__ uint64_t list[kMostCandidates], cum[kMostCandidates];   // cum: weight up to and including
  __shared__ uint64_t wave_sum[kFinalThreads / 64], answer[4];
  __shared__ unsigned long long kept_m;
  const float2 range = row_range(P, row);
  if (!live(range.x)) {
    if (t == 0) {
      P.tokens[row] = -1;
      if (P.probs) P.probs[row] = 0.0f;
    }
    return;
  }
  const RowScale S(P, row, range.x, range.y);
  cumulate<kFinalThreads>(R, B);
  const Cuts C(P, row, S, B);
  const uint32_t n = R.candidates;
  const bool fits = n <= (uint32_t)kMostCandidates;
  if (t == 0) kept_m = 0;
  __syncthreads();
  int size = 2;
  if (fits) {
    while (size < (int)n) size <<= 1;
    for (int i = t; i < size; i += kFinalThreads) list[i] = i < (int)n ? R.list[i] : 0;
    __syncthreads();
    sort_descending(list, size);
    // cumulative weights: those of the whole bins that were not gathered come in between
    constexpr int PER = kMostCandidates / kFinalThreads;
    uint64_t w[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = t * PER + k;
      if (i < (int)n) sum += S.mass_of(S.z_of(of_key((uint32_t)(list[i] >> 32))));
      w[k] = sum;
    }
    uint64_t incl = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_up((unsigned long long)incl, d);
      if ((t & 63) >= d) incl += o;
    }
    if ((t & 63) == 63) wave_sum[t >> 6] = incl;
    __syncthreads();
    uint64_t before = incl - sum;
    for (int v = 0; v < (t >> 6); v++) before += wave_sum[v];
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (t * PER + k < (int)n) cum[t * PER + k] = before + w[k];
    __syncthreads();
    uint64_t full[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = t * PER + k;
      if (i >= (int)n) continue;
      const int b = S.bin_of(S.z_of(of_key((uint32_t)(list[i] >> 32))));
      // the first candidate of this bin: bins are whole in the list
      int lo = 0, hi = i;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (S.bin_of(S.z_of(of_key((uint32_t)(list[mid] >> 32)))) >= b) hi = mid;
        else lo = mid + 1;
      }
      full[k] = B.mass[b] + cum[i] - (lo > 0 ? cum[lo - 1] : 0);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; k++)
      if (t * PER + k < (int)n) cum[t * PER + k] = full[k];
    __syncthreads();
  }
  auto bin_at = [&](int i) { return S.bin_of(S.z_of(of_key((uint32_t)(list[i] >> 32)))); };
  // first candidate from bin `b` on that satisfies a monotone condition on the cumulative weight
  auto first_in = [&](int b, auto cond) {
    int lo = 0, hi = (int)n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const int bm = bin_at(mid);
      if (bm > b || (bm == b && cond(mid))) hi = mid;
      else lo = mid + 1;
    }
    return lo < (int)n ? lo : (int)n - 1;
  };
  // ---- top-k
  uint64_t k_mass = C.k_mass;
  if (C.k_bin >= 0) {
    if (fits) {
      const int start = first_in(C.k_bin, [&](int) { return true; });
      k_mass = cum[start + (int)(C.k - B.count[C.k_bin]) - 1];
    } else {
      k_mass = search_digits<T>(P, row, S, B, C.k_bin, C.k_bin, 0, C.k, 0.0, cum, (uint32_t*)list, answer).mass;
    }
  }
  uint64_t kept = k_mass;
  // ---- top-p
  if (C.use_p) {
    const double target = C.p * (double)k_mass;
    const int b = bin_at_least(B, target);
    uint64_t mass;
    if (b == kBins - 1) mass = B.mass[kBins];
    else if (fits) mass = cum[first_in(b, [&](int i) { return (double)cum[i] >= target; })];
    else mass = search_digits<T>(P, row, S, B, b, b, 1, 0, target, cum, (uint32_t*)list, answer).mass;
    kept = min(kept, mass);
  }
  // ---- min-p: the weights of the interval's elements that pass
  if (C.use_m) {
    uint64_t some = 0;
    auto add = [&](float x) {
      const double z = S.z_of(x);
      const int b = S.bin_of(z);
      if (b >= C.m_lo && b <= C.m_hi && b < kBins - 1 && (z == 0.0 || S.weight_of(z) >= C.min_p)) some += S.mass_of(z);
    };
    if (fits) {
      for (int i = t; i < (int)n; i += kFinalThreads) add(of_key((uint32_t)(list[i] >> 32)));
    } else {
      for (int64_t i = t; i < P.vocab; i += kFinalThreads) {
        const float x = logit<T>(P, row, i);
        if (live(x)) add(x);
      }
    }
    if (some) atomicAdd(&kept_m, (unsigned long long)some);
    __syncthreads();
    // a min_p above 1 keeps the first alone
    const uint64_t mass = C.min_p > 1.0 ? (uint64_t)kUnit : B.mass[C.m_lo] + (uint64_t)kept_m;
    kept = min(kept, mass);
  }
  // ---- the token
  const double target = C.u * (double)kept;
  const int b = bin_above(B, target);
  uint64_t key;
  if (fits) key = list[first_in(b, [&](int i) { return (double)cum[i] > target; })];
  else key = search_digits<T>(P, row, S, B, b, b, 2, 0, target, cum, (uint32_t*)list, answer).key;
  if (t == 0) {
    P.tokens[row] = (int64_t)(uint32_t)~(uint32_t)key;
    if (P.probs) P.probs[row] = (float)(S.weight_of(S.z_of(of_key((uint32_t)(key >> 32)))) * kUnit / (double)kept);
  }
}

// Chunks of a row: enough workgroups for the chip, at least 1024 logits each.
static int sample_chunks(int64_t rows, int64_t vocab) {
  int64_t c = (vocab + 1023) / 1024;
  const int64_t fill = (4 * 256 + rows - 1) / rows;
  if (c > fill) c = fill;
  if (c > kMostChunks) c = kMostChunks;
  return c < 1 ? 1 : (int)c;
}

template <typename T>
static int launch_sample(const SampleParams& P, int64_t rows, hipStream_t st) {
  const dim3 grid((unsigned)P.chunks, (unsigned)rows), block(256);
  hipLaunchKernelGGL((sample_range_kernel<T>), grid, block, 0, st, P);
  int rc = check_launch("sample_rows");
  if (rc) return rc;
  hipLaunchKernelGGL((sample_bins_kernel<T>), grid, block, 0, st, P);
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
  P.logits = logits; P.row_stride = row_stride; P.vocab = vocab;
  P.uniforms = uniforms; P.temperature = temperature; P.top_k = top_k; P.top_p = top_p; P.min_p = min_p;
  P.rows = reinterpret_cast<SampleRow*>(scratch);
  P.chunks = sample_chunks(rows, vocab);
  P.chunk = (int)(((vocab + P.chunks - 1) / P.chunks + 7) / 8 * 8);
  P.tokens = tokens; P.probs = probs;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == TT_F16) return launch_sample<f16_t>(P, rows, st);
  if (dtype == TT_BF16) return launch_sample<bf16_t>(P, rows, st);
  return launch_sample<float>(P, rows, st);
}
