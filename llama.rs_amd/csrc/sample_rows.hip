// sample_rows.hip — one token per row of logits: temperature, top-k, top-p
// and min-p from given random numbers.
#include <math.h>

#include "paged_device.h"
#include "serve_check.h"

namespace rlh {
namespace {

// Two launches. The first reads the logits once: chunks of 4096 values, of
// each its largest key, its mass relative to that, the largest key of every
// 64 values, and, where a row's options may keep many tokens, a histogram of
// counts and masses over eighths of a power of two. The second has a block
// per row and, as a rule, reads only the groups of 64 that can hold a token
// next to the border of what is kept:
//   top-k (small k): the k-th largest of the groups' maxima is at most the
//     k-th largest value, so only groups that reach it are read
//   else: the histogram names the bin that holds the border; its values are
//     sorted, all above are kept
// and then draws: over the list itself, or over the chunks' kept masses and
// inside the one chunk that the draw falls into. A border bin (or list) of
// more than kCand values takes a search over the whole row instead.
constexpr int kMassBits = 42;  // masses in histograms: multiples of 2^-42 of a chunk's largest weight
constexpr uint64_t kMaxRow = 1ull << 21;
constexpr uint64_t kMaxRows = 1ull << 21;
constexpr uint32_t kChunk = 4096;
constexpr uint32_t kGroup = 64;
constexpr uint32_t kBins = 384;        // 48 powers of two; the last one takes the rest
constexpr int kScanThreads = 256;
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kCand = 2048;       // values sorted in LDS
constexpr uint32_t kRadix = 2048;
constexpr uint32_t kListK = 1024;      // largest top-k that takes the groups' maxima

// Ascending as the values are; NaN (either sign) and -infinity give 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 equals 0
  if (!(x > -INFINITY)) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^y for y <= 0 (0 below 2^-1000, NaN and -infinity): Taylor's polynomial of
// degree 11 of 2^f, |f| <= 1/2, off by less than 2^-47.
__device__ __forceinline__ double exp2_neg(double y) {
  const double n = rint(y);
  const double f = (y - n) * 0.6931471805599453;
  double p = 1.0 / 39916800.0;
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return y > -1000.0 ? ldexp(p, (int)n) : 0.0;
}

// exp((x - top) / temperature) with `c` = log2(e) / temperature; 1 at the top
// itself (so infinite tops share the mass), 0 for what has none.
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t top_key, double top, double c) {
  if (key == top_key) return 1.0;
  return key == 0u ? 0.0 : exp2_neg(((double)value_of(key) - top) * c);
}
__device__ __forceinline__ uint64_t mass_of(double w) { return (uint64_t)(w * (double)(1ull << kMassBits) + 0.5); }

// Bin of a value below a row's or a chunk's largest (`base`: its edge
// number): eighths of a power of two, from the top.
__device__ __forceinline__ double edge_of(uint32_t key, double c) { return floor((double)value_of(key) * c * 8.0); }
__device__ __forceinline__ uint32_t bin_of(uint32_t key, uint32_t top_key, double base, double c) {
  if (key == top_key) return 0u;
  const double d = base - edge_of(key, c);
  return key != 0u && d < (double)(kBins - 1) ? (uint32_t)d : kBins - 1;
}

// What a row's options ask for.
struct RowPlan {
  bool greedy, by_k, by_p, list, bins, mass;
  double c, min_p;
};
__device__ __forceinline__ RowPlan row_plan(const rlh_row_sampling& o, uint32_t n) {
  RowPlan r;
  r.greedy = !(o.temperature > 0.0f);
  r.by_k = o.top_k > 0 && o.top_k < n;
  r.by_p = o.top_p > 0.0f && o.top_p < 1.0f;
  r.min_p = o.min_p > 0.0f ? (double)o.min_p : 0.0;
  r.list = r.by_k && o.top_k <= kListK && o.top_k <= n / (2 * kGroup);
  r.bins = !r.greedy && !r.list && (r.by_k || r.by_p || r.min_p > 0.0);
  r.mass = !r.greedy && (r.by_p || !r.list);
  r.c = 1.4426950408889634 / (double)o.temperature;
  return r;
}

// Where a row's intermediate results lie.
struct RowSpace {
  uint32_t* group;   // [groups]
  uint32_t* top;     // [chunks]
  double* mass;      // [chunks]
  uint32_t* count;   // [chunks][kBins]
  uint64_t* bin;     // [chunks][kBins]
};
struct Space {
  uint8_t* base;
  uint64_t row_bytes;
  uint32_t chunks, groups;
  __host__ __device__ RowSpace row(uint64_t r) const {
    uint8_t* p = base + r * row_bytes;
    RowSpace s;
    s.bin = (uint64_t*)p;
    s.mass = (double*)(p + (uint64_t)chunks * kBins * 8);
    s.count = (uint32_t*)(p + (uint64_t)chunks * (kBins * 8 + 8));
    s.top = s.count + (uint64_t)chunks * kBins;
    s.group = s.top + chunks;
    return s;
  }
};

// A row's values are counted from the 16-byte line that its first one lies
// in: value v of the lines is value v - shift of the row.
template <typename T>
struct Row {
  const T* x;
  uint32_t n, shift;
  __device__ __forceinline__ Row(const T* logits, uint64_t stride, uint32_t n_, uint32_t r) {
    x = logits + (size_t)r * stride;
    n = n_;
    shift = (uint32_t)((uintptr_t)x & 15) / sizeof(T);
  }
  __device__ __forceinline__ uint32_t lines() const { return n + shift; }
  __device__ __forceinline__ uint32_t key(uint32_t v) const {
    return v >= shift && v < shift + n ? key_of((float)x[v - shift]) : 0u;
  }
  // the 16 / sizeof(T) keys from v on (v a multiple of that)
  template <int V>
  __device__ __forceinline__ void keys(uint32_t v, uint32_t (&k)[V]) const {
    typedef T TV __attribute__((ext_vector_type(V)));
    if (v >= shift && v + V <= shift + n) {
      const TV a = *(const TV*)(x + ((size_t)v - shift));
#pragma unroll
      for (int i = 0; i < V; i++) k[i] = key_of((float)a[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) k[i] = key(v + i);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kScanThreads) k_sample_scan(const T* logits, uint32_t n, uint64_t stride,
                                                             const rlh_row_sampling* options, Space space) {
  constexpr int V = 16 / sizeof(T);
  constexpr int N = kChunk / kScanThreads / V;  // lines per thread
  constexpr int kGroupLanes = kGroup / V;
  __shared__ uint32_t count[kBins];
  __shared__ uint64_t bin[kBins];
  __shared__ uint32_t tops[kScanThreads / 64];
  __shared__ double sums[kScanThreads / 64];
  const uint32_t t = threadIdx.x, chunk = blockIdx.x % space.chunks, r = blockIdx.x / space.chunks;
  const RowPlan plan = row_plan(options[r], n);
  const RowSpace rs = space.row(r);
  const Row<T> row(logits, stride, n, r);
  if (plan.bins) {
    for (uint32_t i = t; i < kBins; i += kScanThreads) {
      count[i] = 0;
      bin[i] = 0;
    }
  }
  uint32_t k[N][V], top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) row.keys(chunk * kChunk + (i * kScanThreads + t) * V, k[i]);
#pragma unroll
  for (int i = 0; i < N; i++) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < V; e++) m = max(m, k[i][e]);
#pragma unroll
    for (int d = 1; d < kGroupLanes; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    const uint32_t g = (chunk * kChunk + (i * kScanThreads + t) * V) / kGroup;
    if (t % kGroupLanes == 0 && g < space.groups) rs.group[g] = m;
    top = max(top, m);
  }
#pragma unroll
  for (int d = kGroupLanes; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if ((t & 63) == 0) tops[t >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kScanThreads / 64; i++) top = max(top, tops[i]);
  if (t == 0) rs.top[chunk] = top;
  if (!plan.mass) return;
  const double tv = (double)value_of(top), base = edge_of(top, plan.c);
  double sum = 0.0;
  if (top != 0u) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const double w = weight_of(k[i][e], top, tv, plan.c);
        sum += w;
        if (plan.bins && k[i][e] != 0u) {
          const uint32_t b = bin_of(k[i][e], top, base, plan.c);
          atomicAdd(&count[b], 1u);
          atomicAdd((unsigned long long*)&bin[b], (unsigned long long)mass_of(w));
        }
      }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  if ((t & 63) == 0) sums[t >> 6] = sum;
  __syncthreads();
  if (t == 0) rs.mass[chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  if (plan.bins)
    for (uint32_t i = t; i < kBins; i += kScanThreads) {
      rs.count[(uint64_t)chunk * kBins + i] = count[i];
      rs.bin[(uint64_t)chunk * kBins + i] = bin[i];
    }
}

// ---- block-wide sums and searches ---------------------------------------------------
template <typename T>
__device__ __forceinline__ T shfl_up_t(T v, int d) {
  return __shfl_up(v, d);
}
__device__ __forceinline__ uint64_t shfl_up_t(uint64_t v, int d) { return __shfl_up((unsigned long long)v, d); }

struct PickShared {
  uint64_t sorted[kCand];     // (key, ~index), later sorted
  uint32_t key[kCand];        // in index order
  uint32_t index[kCand];
  union {
    uint32_t list[kCand];     // groups that are read
    uint32_t hist[kRadix];
    uint64_t mhist[kRadix];
  };
  double slots[kWaves];
  uint64_t slots64[kWaves];
  uint32_t slots32[kWaves];
  double bcast;
  uint64_t bcast64;
  uint32_t where[4];
};

// Inclusive sum of one value per thread in thread order; *all: the whole.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* slots, T* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = shfl_up_t(x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) slots[wave] = x;
  __syncthreads();
  T off = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    if (i < wave) off += slots[i];
    sum += slots[i];
  }
  *all = sum;
  return off + x;
}

// The k-th largest of f(0..n-1) (k >= 1; 0 when fewer are above 0) by radix
// descent, 11, 11 and 10 bits.
template <typename F>
__device__ uint32_t kth_largest(PickShared& sh, uint32_t n, uint32_t k, F f) {
  const uint32_t t = threadIdx.x;
  uint32_t key = 0, above = 0;
  for (int r = 0; r < 3; r++) {
    const int shift = r == 0 ? 21 : r == 1 ? 10 : 0;
    const uint32_t mask = r == 0 ? 0u : r == 1 ? 0xffe00000u : 0xfffffc00u;
    __syncthreads();
    for (uint32_t i = t; i < kRadix; i += kThreads) sh.hist[i] = 0;
    if (t == 0) sh.where[0] = 0xffffffffu;
    __syncthreads();
    for (uint32_t i = t; i < n; i += kThreads) {
      const uint32_t v = f(i);
      if (v != 0u && ((v ^ key) & mask) == 0) atomicAdd(&sh.hist[(v >> shift) & (r == 2 ? 1023u : 2047u)], 1u);
    }
    __syncthreads();
    // two bins per thread, from the top
    const uint32_t hi = kRadix - 1 - 2 * t, a = sh.hist[hi], b = sh.hist[hi - 1];
    uint32_t all;
    const uint32_t upto = above + block_scan<uint32_t>(a + b, sh.slots32, &all);
    const uint32_t before = upto - a - b;
    if (before < k && upto >= k) {
      const bool first = before + a >= k;
      sh.where[0] = first ? hi : hi - 1;
      sh.where[1] = first ? before : before + a;
    }
    __syncthreads();
    if (sh.where[0] == 0xffffffffu) return 0;
    key |= sh.where[0] << shift;
    above = sh.where[1];
  }
  return key;
}

// Every value with key in [lo, hi] into sh.key / sh.index, in index order;
// false when there are more than kCand. Reads the groups that reach lo.
template <typename T>
__device__ bool gather(PickShared& sh, const Row<T>& row, const RowSpace& rs, uint32_t groups, uint32_t lo, uint32_t hi,
                       uint32_t* count) {
  constexpr int V = 16 / sizeof(T);
  constexpr int kLanes = kGroup / V, kPer = 64 / kLanes;  // lanes of a group, groups of a wave
  const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint32_t found = 0;
  // in rounds of as many groups as the list holds
  for (uint32_t g0 = 0; g0 < groups;) {
    uint32_t listed = 0;
    while (g0 < groups && listed + kThreads <= kCand) {
      const uint32_t g = g0 + t;
      const uint32_t yes = g < groups && rs.group[g] >= lo ? 1u : 0u;
      uint32_t all;
      const uint32_t at = listed + block_scan<uint32_t>(yes, sh.slots32, &all) - yes;
      if (yes) sh.list[at] = g;
      listed += all;
      g0 += kThreads;
    }
    __syncthreads();
    // which values of each group: a bit per value
    for (uint32_t i0 = wave * kPer; i0 < listed; i0 += kWaves * kPer) {
      const uint32_t i = i0 + lane / kLanes;
      uint64_t bits = 0;
      if (i < listed) {
        uint32_t k[V];
        const uint32_t g = sh.list[i];
        row.keys(g * kGroup + lane % kLanes * V, k);
#pragma unroll
        for (int e = 0; e < V; e++) bits |= (uint64_t)(k[e] >= lo && k[e] <= hi) << e;
        bits <<= lane % kLanes * V;
      }
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) bits |= __shfl_xor((unsigned long long)bits, d);
      if (i < listed && lane % kLanes == 0) sh.sorted[i] = bits;
    }
    __syncthreads();
    // places of their values
    for (uint32_t i0 = 0; i0 < listed; i0 += kThreads) {
      const uint32_t i = i0 + t;
      const uint64_t bits = i < listed ? sh.sorted[i] : 0;
      uint32_t all;
      uint32_t at = found + block_scan<uint32_t>((uint32_t)__popcll(bits), sh.slots32, &all) - (uint32_t)__popcll(bits);
      const uint32_t g = i < listed ? sh.list[i] : 0;
      for (uint64_t left = bits; left; left &= left - 1, at++)
        if (at < kCand) sh.index[at] = g * kGroup + (uint32_t)__builtin_ctzll(left);
      found += all;
    }
    __syncthreads();
    if (found > kCand) return false;
  }
  for (uint32_t i = t; i < found; i += kThreads) sh.key[i] = row.key(sh.index[i]);
  __syncthreads();
  *count = found;
  return true;
}

// sh.sorted = the gathered values, key descending and index ascending.
__device__ void sort_gathered(PickShared& sh, uint32_t m) {
  const uint32_t t = threadIdx.x;
  uint32_t P = 2;
  while (P < m) P <<= 1;
  for (uint32_t i = t; i < P; i += kThreads)
    sh.sorted[i] = i < m ? (uint64_t)sh.key[i] << 32 | (uint32_t)~sh.index[i] : 0ull;
  __syncthreads();
  if (P <= 64) {  // one wave, in registers
    if (t < 64) {
      uint64_t k = t < P ? sh.sorted[t] : 0ull;
      for (uint32_t size = 2; size <= P; size <<= 1)
        for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
          const uint64_t o = __shfl_xor((unsigned long long)k, (int)stride);
          const bool larger = ((t & size) == 0) == ((t & stride) == 0);
          k = (k > o) == larger ? k : o;
        }
      if (t < P) sh.sorted[t] = k;
    }
    __syncthreads();
    return;
  }
  for (uint32_t size = 2; size <= P; size <<= 1)
    for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
      for (uint32_t q = t; q < P / 2; q += kThreads) {
        const uint32_t i = 2 * stride * (q / stride) + q % stride, j = i + stride;
        const bool desc = (i & size) == 0;
        const uint64_t a = sh.sorted[i], b = sh.sorted[j];
        if ((a < b) == desc) {
          sh.sorted[i] = b;
          sh.sorted[j] = a;
        }
      }
      __syncthreads();
    }
}

// The border: kept are keys above `key` and, of equal ones, indices up to `index`.
struct Border {
  uint32_t key, index;
};
__device__ __forceinline__ bool kept(const Border& b, uint32_t key, uint32_t index) {
  return key > b.key || (key == b.key && index <= b.index);
}

// The border within the sorted values: `k` more by count, mass up to goal_p
// on top of `above`, weights of at least min_p; none of the three reached:
// the last one. `force`: the first of them is the row's first, always kept.
__device__ Border cut_sorted(PickShared& sh, uint32_t m, const RowPlan& plan, uint32_t k, double above, double goal_p,
                             uint32_t top_key, bool force) {
  const uint32_t t = threadIdx.x;
  const double top = (double)value_of(top_key);
  if (t == 0) sh.where[0] = m;  // values kept
  __syncthreads();
  double run = above;
  for (uint32_t i0 = 0; i0 < m; i0 += kThreads) {
    const uint32_t i = i0 + t;
    const double w = i < m ? weight_of((uint32_t)(sh.sorted[i] >> 32), top_key, top, plan.c) : 0.0;
    double all;
    const double upto = run + block_scan<double>(w, sh.slots, &all);
    // dropped: past k, reached before it, or too light
    if (i < m && (i >= k || (plan.by_p && upto - w >= goal_p) || w < plan.min_p) && !(force && i == 0))
      atomicMin(&sh.where[0], i);
    run += all;
    __syncthreads();
  }
  const uint32_t n = sh.where[0];
  __syncthreads();
  if (n == 0) return Border{0xffffffffu, 0u};
  const uint64_t last = sh.sorted[n - 1];
  return Border{(uint32_t)(last >> 32), ~(uint32_t)last};
}

// The border by a search over the whole row: radix descent on counts and on
// masses (whole numbers, so their order does not matter) side by side.
template <typename T>
__device__ Border search_row(PickShared& sh, const Row<T>& row, const RowPlan& plan, uint32_t goal_k, double share_p,
                             uint32_t top_key) {
  const uint32_t t = threadIdx.x;
  const double top = (double)value_of(top_key);
  const uint32_t lines = row.lines();
  Border border{1u, 0xffffffffu};
  auto nth_equal = [&](uint32_t key, uint32_t nth) {  // index of the nth (from 1) value that equals key
    uint32_t seen = 0;
    for (uint32_t v0 = 0; v0 < lines; v0 += kThreads) {
      const uint32_t v = v0 + t, yes = v < lines && row.key(v) == key ? 1u : 0u;
      uint32_t all;
      const uint32_t upto = seen + block_scan<uint32_t>(yes, sh.slots32, &all);
      if (yes && upto == nth) sh.where[2] = v;
      seen += all;
      if (seen >= nth) break;
    }
    __syncthreads();
    return sh.where[2];
  };
  auto tighten = [&](uint32_t key, uint32_t index) {
    if (key > border.key || (key == border.key && index < border.index)) border = Border{key, index};
  };
  if (plan.by_k) {
    const uint32_t key = kth_largest(sh, lines, goal_k, [&](uint32_t v) { return row.key(v); });
    if (key != 0u) {
      uint32_t part = 0, above = 0;
      for (uint32_t v = t; v < lines; v += kThreads) part += row.key(v) > key ? 1u : 0u;
      block_scan<uint32_t>(part, sh.slots32, &above);
      __syncthreads();
      tighten(key, nth_equal(key, goal_k - above));
    }
  }
  if (plan.by_p) {
    uint64_t part = 0, sum = 0;
    for (uint32_t v = t; v < lines; v += kThreads) part += mass_of(weight_of(row.key(v), top_key, top, plan.c));
    block_scan<uint64_t>(part, sh.slots64, &sum);
    const double goal = share_p * (double)sum;
    uint32_t key = 0;
    uint64_t above = 0;
    for (int r = 0; r < 3; r++) {
      const int shift = r == 0 ? 21 : r == 1 ? 10 : 0;
      const uint32_t mask = r == 0 ? 0u : r == 1 ? 0xffe00000u : 0xfffffc00u;
      __syncthreads();
      for (uint32_t i = t; i < kRadix; i += kThreads) sh.mhist[i] = 0;
      if (t == 0) sh.where[0] = 0;
      __syncthreads();
      for (uint32_t v = t; v < lines; v += kThreads) {
        const uint32_t k = row.key(v);
        if (k != 0u && ((k ^ key) & mask) == 0)
          atomicAdd((unsigned long long*)&sh.mhist[(k >> shift) & (r == 2 ? 1023u : 2047u)],
                    (unsigned long long)mass_of(weight_of(k, top_key, top, plan.c)));
      }
      __syncthreads();
      const uint32_t hi = kRadix - 1 - 2 * t;
      const uint64_t a = sh.mhist[hi], b = sh.mhist[hi - 1];
      uint64_t all;
      const uint64_t upto = above + block_scan<uint64_t>(a + b, sh.slots64, &all);
      const uint64_t before = upto - a - b;
      auto reached = [&](uint64_t v) { return v > 0 && (double)v >= goal; };
      if (!reached(before) && reached(upto)) {
        const bool first = reached(before + a);
        sh.where[0] = first ? hi : hi - 1;
        sh.bcast64 = first ? before : before + a;
      }
      __syncthreads();
      key |= sh.where[0] << shift;
      above = sh.bcast64;
    }
    const uint64_t w = mass_of(weight_of(key, top_key, top, plan.c));
    uint32_t nth = 1;
    if (w > 0) {
      const double d = (goal - (double)above) / (double)w;
      nth = d > 1.0 ? (uint32_t)fmin(d, (double)kMaxRow) : 1u;
      while (nth > 1 && (double)(above + (uint64_t)(nth - 1) * w) >= goal) nth--;
      while ((double)(above + (uint64_t)nth * w) < goal && nth < row.n) nth++;
    }
    tighten(key, nth_equal(key, nth));
  }
  if (plan.min_p > 0.0) {
    // the lightest key that still has min_p (the first is kept whatever it has)
    uint32_t lo = 1, hi = top_key;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (weight_of(mid, top_key, top, plan.c) >= plan.min_p)
        hi = mid;
      else
        lo = mid + 1;
    }
    if (weight_of(top_key, top_key, top, plan.c) < plan.min_p)
      tighten(top_key, nth_equal(top_key, 1));
    else
      tighten(lo, 0xffffffffu);
  }
  return border;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_pick(const T* logits, uint32_t n, uint64_t stride,
                                                          const rlh_row_sampling* options, const float* us,
                                                          uint32_t* tokens, Space space) {
  __shared__ PickShared sh;
  const uint32_t t = threadIdx.x, r = blockIdx.x, lane = t & 63, wave = t >> 6;
  const rlh_row_sampling o = options[r];
  const RowPlan plan = row_plan(o, n);
  const RowSpace rs = space.row(r);
  const Row<T> row(logits, stride, n, r);
  const uint32_t chunks = (row.lines() + kChunk - 1) / kChunk, groups = (row.lines() + kGroup - 1) / kGroup;
  uint32_t top_key = 0;
  for (uint32_t i = t; i < chunks; i += kThreads) top_key = max(top_key, rs.top[i]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top_key = max(top_key, (uint32_t)__shfl_xor((int)top_key, d));
  if (lane == 0) sh.slots32[wave] = top_key;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) top_key = max(top_key, sh.slots32[i]);
  __syncthreads();
  if (top_key == 0u) {
    if (t == 0) tokens[r] = 0;
    return;
  }
  if (plan.greedy) {
    // the first group that holds it, the first of its values
    if (t == 0) sh.where[0] = 0xffffffffu;
    __syncthreads();
    for (uint32_t g = t; g < groups; g += kThreads)
      if (rs.group[g] == top_key) {
        atomicMin(&sh.where[0], g);
        break;
      }
    __syncthreads();
    if (wave == 0) {
      const uint32_t v = sh.where[0] * kGroup + lane;
      const uint64_t hit = __ballot(row.key(v) == top_key);
      if (lane == 0) tokens[r] = sh.where[0] * kGroup + (uint32_t)__builtin_ctzll(hit) - row.shift;
    }
    return;
  }
  const double top = (double)value_of(top_key);
  // masses of chunks are relative to their own largest weight
  auto chunk_factor = [&](uint32_t ch) { return weight_of(rs.top[ch], top_key, top, plan.c); };
  double sum = 0.0;
  if (plan.mass) {
    double part = 0.0;
    for (uint32_t i = t; i < chunks; i += kThreads) part += chunk_factor(i) * rs.mass[i];
    block_scan<double>(part, sh.slots, &sum);
    __syncthreads();
  }
  const double goal_p = (double)o.top_p * sum;
  const float u = us[r];
  const double uu = u > 0.0f ? fmin((double)u, 1.0) : 0.0;

  Border border{0u, 0xffffffffu};  // everything
  uint32_t border_bin = kBins, gathered = 0;  // the bin that holds it, and its values in sh.key / sh.index
  if (plan.list) {
    const uint32_t lo = max(kth_largest(sh, groups, o.top_k, [&](uint32_t g) { return rs.group[g]; }), 1u);
    uint32_t m;
    if (gather(sh, row, rs, groups, lo, 0xffffffffu, &m)) {
      sort_gathered(sh, m);
      border = cut_sorted(sh, m, plan, o.top_k, 0.0, goal_p, top_key, true);
      // the draw over the list, which is in index order
      double total = 0.0;
      double w[kCand / kThreads];
#pragma unroll
      for (uint32_t j = 0; j < kCand / kThreads; j++) {
        const uint32_t i = t * (kCand / kThreads) + j;
        w[j] = i < m && kept(border, sh.key[i], sh.index[i]) ? weight_of(sh.key[i], top_key, top, plan.c) : 0.0;
        total += w[j];
      }
      double all;
      double run = block_scan<double>(total, sh.slots, &all) - total;
      const double goal = uu * all;
      if (t == 0) sh.where[3] = 0xffffffffu;
      __syncthreads();
#pragma unroll
      for (uint32_t j = 0; j < kCand / kThreads; j++) {
        run += w[j];
        if (w[j] > 0.0 && run > goal) atomicMin(&sh.where[3], t * (kCand / kThreads) + j);
      }
      __syncthreads();
      if (sh.where[3] == 0xffffffffu) {  // u at its upper end: the last one with mass
        if (t == 0) sh.where[2] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kCand / kThreads; j++)
          if (w[j] > 0.0) atomicMax(&sh.where[2], t * (kCand / kThreads) + j);
        __syncthreads();
        if (t == 0) tokens[r] = sh.index[sh.where[2]] - row.shift;
        return;
      }
      if (t == 0) tokens[r] = sh.index[sh.where[3]] - row.shift;
      return;
    }
    border = search_row(sh, row, plan, o.top_k, (double)o.top_p, top_key);
  } else if (plan.bins) {
    // the row's histogram, one bin per thread, chunk after chunk
    const double base = edge_of(top_key, plan.c);
    uint32_t cnt = 0;
    double mass = 0.0;
    if (t < kBins) {
      for (uint32_t ch = 0; ch < chunks; ch++) {
        const uint32_t ck = rs.top[ch];
        if (ck == 0u) continue;
        const uint32_t off = bin_of(ck, top_key, base, plan.c);
        if (t < off) continue;
        if (t < kBins - 1) {
          cnt += rs.count[(uint64_t)ch * kBins + t - off];
          mass += chunk_factor(ch) * (double)rs.bin[(uint64_t)ch * kBins + t - off];
        }
      }
    }
    mass *= 1.0 / (double)(1ull << kMassBits);
    uint32_t all32;
    double alld;
    const uint32_t upto_k = block_scan<uint32_t>(cnt, sh.slots32, &all32);
    const double upto_p = block_scan<double>(mass, sh.slots, &alld);
    if (t == 0) sh.where[0] = kBins - 1;
    __syncthreads();
    // the first bin at which one of the three ends
    uint32_t min_bin = kBins;
    if (plan.min_p > 0.0) {
      // (NaN: an infinite top, whose bin holds all that have mass)
      const double d = base - floor((top * plan.c + log2(fmin(plan.min_p, 1.0))) * 8.0);
      min_bin = d >= (double)(kBins - 1) ? kBins : d > 0.0 ? (uint32_t)d : 0u;
    }
    if (t < kBins - 1 &&
        ((plan.by_k && upto_k >= o.top_k) || (plan.by_p && upto_p >= goal_p) || t >= min_bin))
      atomicMin(&sh.where[0], t);
    __syncthreads();
    const uint32_t bin = sh.where[0];
    __syncthreads();
    if (t == bin) {
      sh.where[1] = upto_k - cnt;
      sh.bcast = upto_p - mass;
    }
    __syncthreads();
    const uint32_t above_k = sh.where[1];
    const double above_p = sh.bcast;
    if (bin < kBins - 1) {
      // the bin's keys: bins fall as keys rise
      auto first_key = [&](uint32_t b) {  // the least key of bin b or above
        uint32_t lo = 1, hi = top_key;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo) / 2;
          if (bin_of(mid, top_key, base, plan.c) <= b)
            hi = mid;
          else
            lo = mid + 1;
        }
        return lo;
      };
      if (t < 2) sh.where[2 + t] = t == 0 ? first_key(bin) : bin == 0 ? top_key + 1 : first_key(bin - 1);
      __syncthreads();
      const uint32_t lo = sh.where[2], hi = sh.where[3] - 1;
      uint32_t m;
      if (gather(sh, row, rs, groups, lo, hi, &m)) {
        sort_gathered(sh, m);
        border = cut_sorted(sh, m, plan, plan.by_k ? o.top_k - above_k : 0xffffffffu, above_p, goal_p, top_key, bin == 0);
        if (border.key == 0xffffffffu) border = Border{hi + 1, 0xffffffffu};  // the bins above, and nothing of this one
        border_bin = bin;
        gathered = m;
      } else {
        border = search_row(sh, row, plan, o.top_k, (double)o.top_p, top_key);
      }
    }
  }
  // the draw over the chunks' kept masses, then within one chunk
  const double base = edge_of(top_key, plan.c);
  auto chunk_kept = [&](uint32_t ch) {  // a whole wave; every lane gets the sum
    double s = 0.0;
    if (border_bin < kBins) {  // the bins above the border's, and what is kept of that one
      const uint32_t off = bin_of(rs.top[ch], top_key, base, plan.c);
      for (uint32_t i = lane; off + i < border_bin; i += 64) s += (double)rs.bin[(uint64_t)ch * kBins + i];
      s *= chunk_factor(ch) * (1.0 / (double)(1ull << kMassBits));
      for (uint32_t i = lane; i < gathered; i += 64)
        if (sh.index[i] / kChunk == ch && kept(border, sh.key[i], sh.index[i])) s += weight_of(sh.key[i], top_key, top, plan.c);
    } else {
      for (uint32_t i = lane; i < kChunk; i += 64) {
        const uint32_t v = ch * kChunk + i, k = row.key(v);
        if (k != 0u && kept(border, k, v)) s += weight_of(k, top_key, top, plan.c);
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    return s;
  };
  __syncthreads();
  double* kept_mass = (double*)sh.sorted;  // [chunks], at most 513
  for (uint32_t ch = wave; ch < chunks; ch += kWaves) {
    const bool some = rs.top[ch] != 0u && rs.top[ch] >= border.key;
    const double s = !some ? 0.0 : border.key == 0u ? chunk_factor(ch) * rs.mass[ch] : chunk_kept(ch);
    if (lane == 0) kept_mass[ch] = s;
  }
  __syncthreads();
  double total = 0.0;
  const double mine = t < chunks ? kept_mass[t] : 0.0;
  const double upto = block_scan<double>(mine, sh.slots, &total);
  const double goal = uu * total;
  if (t == 0) {
    sh.where[0] = 0xffffffffu;
    sh.where[1] = 0;
    sh.where[2] = 0xffffffffu;
    sh.where[3] = 0;
  }
  __syncthreads();
  if (mine > 0.0) {
    if (upto > goal) atomicMin(&sh.where[0], t);
    atomicMax(&sh.where[1], t);
  }
  __syncthreads();
  const uint32_t ch = sh.where[0] != 0xffffffffu ? sh.where[0] : sh.where[1];
  if (t == ch) sh.bcast = upto - mine;
  // consecutive values per thread, so that sums in thread order are in index order
  constexpr uint32_t kPer = kChunk / kThreads;
  double w[kPer], s = 0.0, all;
#pragma unroll
  for (uint32_t j = 0; j < kPer; j++) {
    const uint32_t v = ch * kChunk + t * kPer + j, k = row.key(v);
    w[j] = k != 0u && kept(border, k, v) ? weight_of(k, top_key, top, plan.c) : 0.0;
    s += w[j];
  }
  double run = block_scan<double>(s, sh.slots, &all) - s + sh.bcast;
#pragma unroll
  for (uint32_t j = 0; j < kPer; j++) {
    run += w[j];
    const uint32_t v = ch * kChunk + t * kPer + j;
    if (w[j] > 0.0 && run > goal) atomicMin(&sh.where[2], v);
    if (w[j] >= 0x1p-43) atomicMax(&sh.where[3], v);
  }
  __syncthreads();
  // (none past the goal: u at its upper end, or sums that differ in their last bits)
  if (t == 0) tokens[r] = (sh.where[2] != 0xffffffffu ? sh.where[2] : sh.where[3]) - row.shift;
}

Space sample_space(void* base, uint64_t n) {
  Space s;
  s.base = (uint8_t*)base;
  // a row may begin up to 7 values into its first line
  s.chunks = (uint32_t)((n + 7 + kChunk - 1) / kChunk);
  s.groups = (uint32_t)((n + 7 + kGroup - 1) / kGroup);
  s.row_bytes = ((uint64_t)s.chunks * (kBins * 12 + 12) + (uint64_t)s.groups * 4 + 255) / 256 * 256;
  return s;
}

template <typename T>
void launch_sample(const void* logits, uint64_t n_rows, uint64_t n, uint64_t stride, const rlh_row_sampling* options,
                   const float* u, uint32_t* tokens, const Space& space, hipStream_t s) {
  hipLaunchKernelGGL(k_sample_scan<T>, dim3(space.chunks * (uint32_t)n_rows), dim3(kScanThreads), 0, s, (const T*)logits,
                     (uint32_t)n, stride, options, space);
  hipLaunchKernelGGL(k_sample_pick<T>, dim3((uint32_t)n_rows), dim3(kThreads), 0, s, (const T*)logits, (uint32_t)n,
                     stride, options, u, tokens, space);
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

uint64_t rlh_sample_rows_workspace(uint64_t n_rows, uint64_t n) {
  if (n == 0 || n > kMaxRow || n_rows > kMaxRows) return 0;
  return n_rows * sample_space(nullptr, n).row_bytes;
}

int rlh_sample_rows(uint32_t type, const void* logits, uint64_t n_rows, uint64_t n, uint64_t stride,
                    const rlh_row_sampling* options, const float* u, uint32_t* tokens, void* workspace,
                    uint64_t workspace_bytes, void* stream) {
  const uint32_t size = float_type_size(type);
  if (!size) return serve_error(RLH_EUNSUP, "logits are not F32, F16 or BF16");
  if (n == 0 || n > kMaxRow) return serve_error(RLH_EINVAL, "n outside [1, 2^21]");
  if (n_rows > kMaxRows || n_rows * sample_space(nullptr, n).chunks >= (1ull << 24))
    return serve_error(RLH_EUNSUP, "more than 2^21 rows, or 2^36 logits");
  if (n_rows == 0) return RLH_OK;
  if (!logits) return serve_error(RLH_EINVAL, "logits is null");
  if (!aligned(logits, size)) return serve_error(RLH_EINVAL, "logits is not aligned to its type");
  if (stride < n || stride > (1ull << 32)) return serve_error(RLH_EINVAL, "stride below n or above 2^32");
  if (!options || !u || !tokens) return serve_error(RLH_EINVAL, "null argument");
  if (!aligned(options, 16) || !aligned(u, 4) || !aligned(tokens, 4))
    return serve_error(RLH_EINVAL, "options, u or tokens is misaligned");
  const uint64_t need = rlh_sample_rows_workspace(n_rows, n);
  if (need && !workspace) return serve_error(RLH_EINVAL, "workspace is null");
  if (need > workspace_bytes)
    return serve_error(RLH_EINVAL, "workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(need) + " needed");
  if (need && !aligned(workspace, 16)) return serve_error(RLH_EINVAL, "workspace is not aligned to 16 bytes");
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("logits", logits));
  RLH_TRY(dev("options", options));
  RLH_TRY(dev("u", u));
  RLH_TRY(dev("tokens", tokens));
  if (need) RLH_TRY(dev("workspace", workspace));
  hipStream_t s = (hipStream_t)stream;
  const Space space = sample_space(workspace, n);
  if (type == RLH_TYPE_F32)
    launch_sample<float>(logits, n_rows, n, stride, options, u, tokens, space, s);
  else if (type == RLH_TYPE_F16)
    launch_sample<_Float16>(logits, n_rows, n, stride, options, u, tokens, space, s);
  else
    launch_sample<__bf16>(logits, n_rows, n, stride, options, u, tokens, space, s);
  return launched("rlh_sample_rows");
}

}  // extern "C"
