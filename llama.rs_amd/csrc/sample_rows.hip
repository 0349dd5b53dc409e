// sample_rows.hip — one token per row of logits: temperature, top-k, top-p
// and min-p from given random numbers.
#include <math.h>

#include "paged_device.h"
#include "rlh_device.h"
#include "serve_check.h"

namespace rlh {
namespace {

// Two launches. The first reads the logits once: chunks of 4096 values, of
// each its largest key, its mass relative to that, the largest key of every
// 64 values, and, where a row's options may keep many tokens, a histogram of
// counts and masses over sixteenths of a power of two. The second has a block
// per row and, as a rule, reads only the groups of 64 that can hold a token
// next to the border of what is kept:
//   top-k (small k): the k-th largest of the groups' maxima is at most the
//     k-th largest value, so only groups that reach it are read
//   else: the histogram names the bin that holds the border; only its values
//     are looked at, all above are kept
// A range of keys that holds the border is narrowed by histograms of 2048
// bins until 64 values are left, which one wave sorts. The draw runs over the
// list itself, or over the chunks' kept masses and inside the one chunk that
// it falls into.
// Masses are doubles and integers, so that no order of summing changes them.
// A weight is off by 2^-37 of itself, a value in a bin by 2^-39 more, and
// narrowing rounds each to 2^-43 of the range's largest: a border is where 64
// bits put it to 2^-36 of the mass. What lies below the histogram (2^-39.9 of
// the largest) is searched as one more bin, down to 2^-43; if no bound ends
// there either, the rest is dropped.
// The doubles bound the first launch: 192 rows of 151936 f32 values (117 MB) take 17 to 19 us where
// only maxima are asked for (6.0 TB/s), 33 with masses and 41 with histograms,
// where every SIMD issues vector instructions in 95 % of the cycles (34 and 41
// per value and lane, 18 and 16 of them of doubles).
// The second is bound by chains of loads and block-wide sums from a cold start
// (top-k 40: 17 us) and, where the border lies deep, by what one compute unit
// reads (31 GB/s: a nucleus of 0.9 of a row as normal numbers have it, 54 us).
// 192 rows of options of every kind: 87 us; one row of top-k 40: 21.

constexpr int kMassBits = 42;  // masses within a range: multiples of 2^-42 of the largest weight in it
constexpr double kLeastWeight = 0x1p-43;  // of the largest: a token of less is not taken for the last one
constexpr uint64_t kMaxRow = 1ull << 21;
constexpr uint64_t kMaxRows = 1ull << 21;
constexpr uint32_t kChunk = 4096;
constexpr uint32_t kGroup = 64;
constexpr uint32_t kBins = 640;        // 40 powers of two; the last one takes the rest
constexpr int kScanThreads = 256;
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kCand = 2048;       // values held in LDS
constexpr uint32_t kListed = 2560;     // groups read at a time
constexpr uint32_t kFine = 2048;       // bins of a narrowing step
constexpr uint32_t kListK = 1024;      // largest top-k that takes the groups' maxima

// Ascending as the values are; NaN (either sign) and -infinity give 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 equals 0
  if (!(x > -INFINITY)) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kLeastKey = 0x00800000u, kMostKey = 0xff800000u;  // of the lowest finite value, of infinity
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds, and the sum's low bits are the integer

// 2^y for -1000 <= y <= 0: Taylor's polynomial of degree 9 of 2^f, |f| <= 1/2,
// off by less than 2^-37 (7 10^-12, where two tokens' borders lie 10^-6 of the
// mass apart at best). Rounding, scaling and conversion
// instructions of doubles run at a quarter of the rate of sums and products,
// so y is rounded by adding kRound.
struct Exp2 {
  double round, c9, c8, c7, c6, c5, c4, c3, c2, c1;
};
__device__ __forceinline__ double exp2_within(double y, const Exp2& q) {
  const double z = y + q.round;
  const double f = y - (z - q.round);
  double p = q.c9;
  p = fma(p, f, q.c8);
  p = fma(p, f, q.c7);
  p = fma(p, f, q.c6);
  p = fma(p, f, q.c5);
  p = fma(p, f, q.c4);
  p = fma(p, f, q.c3);
  p = fma(p, f, q.c2);
  p = fma(p, f, q.c1);
  p = fma(p, f, 1.0);
  const uint64_t n = __builtin_bit_cast(uint64_t, z) << 52;  // (negative: the sum wraps as it should)
  return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, p) + n);
}
constexpr double power(double x, int n) { return n ? x * power(x, n - 1) : 1.0; }
constexpr double kLn2 = 0.6931471805599453;
constexpr Exp2 kExp2 = {kRound,
                        power(kLn2, 9) / 362880.0,
                        power(kLn2, 8) / 40320.0,
                        power(kLn2, 7) / 5040.0,
                        power(kLn2, 6) / 720.0,
                        power(kLn2, 5) / 120.0,
                        power(kLn2, 4) / 24.0,
                        power(kLn2, 3) / 6.0,
                        power(kLn2, 2) / 2.0,
                        kLn2};
__device__ __forceinline__ double exp2_within(double y) { return exp2_within(y, kExp2); }
__device__ __forceinline__ double opaque(double x) {
  asm("" : "+s"(x));
  return x;
}
// The same factors in scalar registers, of which the compiler knows no value:
// else it moves each into vector registers before every use.
__device__ __forceinline__ Exp2 exp2_factors() {
  return Exp2{opaque(kExp2.round), opaque(kExp2.c9), opaque(kExp2.c8), opaque(kExp2.c7), opaque(kExp2.c6),
              opaque(kExp2.c5),    opaque(kExp2.c4), opaque(kExp2.c3), opaque(kExp2.c2), opaque(kExp2.c1)};
}
// 0 below 2^-1000, NaN and -infinity.
__device__ __forceinline__ double exp2_neg(double y) { return y > -1000.0 ? exp2_within(y) : 0.0; }

// exp((x - top) / temperature) with `c` = log2(e) / temperature; 1 at the top
// itself (so infinite tops share the mass), 0 for what has none.
__device__ __forceinline__ double weight_of(uint32_t key, uint32_t top_key, double top, double c) {
  if (key == top_key) return 1.0;
  return key == 0u ? 0.0 : exp2_neg(((double)value_of(key) - top) * c);
}
__device__ __noinline__ double weight_called(uint32_t key, uint32_t top_key, double top, double c) {
  return weight_of(key, top_key, top, c);
}
// Bins of a histogram: the value's logarithm of its weight, rounded to
// sixteenths of a power of two and counted from the largest's (`base`) down.
// From 2^51 on, where adding kRound rounds to more than whole numbers, they are
// taken as they are: two f32 values are equal there or 2^27 apart.
constexpr double kLastRounded = 0x1p51;
__device__ __forceinline__ double edge_of(double x16) { return fabs(x16) < kLastRounded ? (x16 + kRound) - kRound : x16; }
__device__ __forceinline__ double edge_of(uint32_t key, double c) { return edge_of((double)value_of(key) * (c * 16.0)); }
__device__ __forceinline__ uint32_t bin_of(uint32_t key, uint32_t top_key, double base, double c) {
  if (key == top_key) return 0u;
  const double d = base - edge_of(key, c);
  return key != 0u && d < (double)(kBins - 1) ? (uint32_t)d : kBins - 1;
}
// Their words: a bin's count from bit 51 on, below it its mass as multiples of
// 2^-38 of the weight at the bin's middle. A value's weight is 2^(-1/32) to
// 2^(1/32) of that, so 4096 of them fit 51 bits, and each is rounded by 2^-39 of itself, however
// small the bin's weights are.
constexpr int kBinShift = 51;
constexpr uint64_t kBinMask = (1ull << kBinShift) - 1;
constexpr double kBinUnit = 0x1p-38;
// 2^(f / 16) for |f| <= 1/2 in those units: Taylor's polynomial of degree 5,
// off by less than 2^-42.
struct BinExp2 {
  double c5, c4, c3, c2, c1, unit, big;
};
__device__ __forceinline__ uint64_t bin_word(double f, const BinExp2& q) {
  double p = q.c5;
  p = fma(p, f, q.c4);
  p = fma(p, f, q.c3);
  p = fma(p, f, q.c2);
  p = fma(p, f, q.c1);
  p = fma(p, f, 1.0);
  // (the low bits of a sum with 2^52 are the rounded integer)
  return (__builtin_bit_cast(uint64_t, fma(p, q.unit, q.big)) & kBinMask) | 1ull << kBinShift;
}
__device__ __forceinline__ BinExp2 bin_factors() {
  constexpr double g = kLn2 / 16.0, c5 = power(g, 5) / 120.0, c4 = power(g, 4) / 24.0, c3 = power(g, 3) / 6.0, c2 = g * g / 2.0;
  return BinExp2{opaque(c5), opaque(c4), opaque(c3), opaque(c2), opaque(g), opaque(1.0 / kBinUnit), opaque(0x1p52)};
}

// A unit of bin b's mass, as a share of the top's weight.
__device__ __forceinline__ double bin_weight(uint32_t b, double base, double top, double c) {
  if (!(top < INFINITY)) return b == 0 ? kBinUnit : 0.0;
  return exp2_neg(((base - (double)b) - top * (c * 16.0)) * (1.0 / 16.0)) * kBinUnit;
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
    s.top = (uint32_t*)(p + (uint64_t)chunks * (kBins * 8 + 8));
    s.group = s.top + chunks;
    return s;
  }
};

constexpr uint32_t kCached = 2560;     // groups whose maxima are held in LDS
constexpr uint32_t kMaxChunks = (uint32_t)(kMaxRow / kChunk) + 1;

// A row's values are counted from the 16-byte line that its first one lies
// in: value v of the lines is value v - shift of the row.
template <typename T>
struct Row {
  // (known to be global memory also in called functions: loads through a
  // generic pointer are counted with LDS reads, which then wait for them)
  const RLH_GLOBAL T* x;
  uint32_t n, shift;
  __device__ __forceinline__ Row(const T* logits, uint64_t stride, uint32_t n_, uint32_t r) {
    x = (const RLH_GLOBAL T*)(logits + (size_t)r * stride);
    n = n_;
    shift = (uint32_t)((uintptr_t)x & 15) / sizeof(T);
  }
  __device__ __forceinline__ uint32_t lines() const { return n + shift; }
  __device__ __forceinline__ uint32_t key(uint32_t v) const {
    return v >= shift && v < shift + n ? key_of((float)x[v - shift]) : 0u;
  }
  // the line at v (a multiple of V); NaN where it lies outside of the row
  static constexpr int V = 16 / sizeof(T);
  typedef T Line __attribute__((ext_vector_type(V)));
  __device__ __forceinline__ Line line(uint32_t v) const {
    Line a;
    if (v >= shift && v + V <= shift + n) {
      a = *(const RLH_GLOBAL Line*)(x + ((size_t)v - shift));
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) a[i] = v + i >= shift && v + i < shift + n ? x[v + i - shift] : (T)__builtin_nanf("");
    }
    return a;
  }
};

// The larger of x and of what lane ^ 1, ^ 2, and then the mirrored lane of 8 or
// 16 hold: after all of them the largest of the lanes.
template <int CTRL>
__device__ __forceinline__ float max_dpp(float x) {
  return fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(__float_as_uint(x), __float_as_uint(x), CTRL, 0xf, 0xf, false)));
}
template <int LANES>
__device__ __forceinline__ float max_of_lanes(float x) {
  x = max_dpp<0xb1>(x);   // quad_perm 1, 0, 3, 2
  x = max_dpp<0x4e>(x);   // quad_perm 2, 3, 0, 1
  x = max_dpp<0x141>(x);  // row_half_mirror
  return LANES == 16 ? max_dpp<0x140>(x) : x;  // row_mirror
}

template <typename T>
__global__ void __launch_bounds__(kScanThreads) k_sample_scan(const T* logits, uint32_t n, uint64_t stride,
                                                             const rlh_row_sampling* options, Space space) {
  constexpr int V = 16 / sizeof(T);
  constexpr int N = kChunk / kScanThreads / V;  // lines per thread
  constexpr int kGroupLanes = kGroup / V;
  __shared__ uint64_t bin[kBins];
  __shared__ uint32_t tops[kScanThreads / 64];
  __shared__ double sums[kScanThreads / 64];
  const uint32_t t = threadIdx.x, chunk = blockIdx.x % space.chunks, r = blockIdx.x / space.chunks;
  const Exp2 exp2 = exp2_factors();
  const BinExp2 bin_exp2 = bin_factors();
  const RowPlan plan = row_plan(options[r], n);
  const RowSpace rs = space.row(r);
  const Row<T> row(logits, stride, n, r);
  if (plan.bins) {
    for (uint32_t i = t; i < kBins; i += kScanThreads) bin[i] = 0;
  }
  typename Row<T>::Line line[N];
  if (chunk * kChunk >= row.shift && (chunk + 1) * kChunk <= row.shift + n) {
    // (all within the row, as most are)
    const RLH_GLOBAL T* x = row.x + ((size_t)chunk * kChunk - row.shift);
#pragma unroll
    for (int i = 0; i < N; i++) line[i] = *(const RLH_GLOBAL typename Row<T>::Line*)(x + (i * kScanThreads + t) * V);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) line[i] = row.line(chunk * kChunk + (i * kScanThreads + t) * V);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    float m = -INFINITY;  // (NaN is not larger)
#pragma unroll
    for (int e = 0; e < V; e++) m = fmaxf(m, (float)line[i][e]);
    const uint32_t km = key_of(max_of_lanes<kGroupLanes>(m));
    const uint32_t g = (chunk * kChunk + (i * kScanThreads + t) * V) / kGroup;
    if (t % kGroupLanes == 0 && g < space.groups) rs.group[g] = km;
    top = max(top, km);
  }
#pragma unroll
  for (int d = kGroupLanes; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if ((t & 63) == 0) tops[t >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kScanThreads / 64; i++) top = max(top, tops[i]);
  top = (uint32_t)__builtin_amdgcn_readfirstlane((int)top);  // (the block's: known to be uniform from here)
  if (t == 0) rs.top[chunk] = top;
  if (!plan.mass) return;
  const double tv = (double)value_of(top), base = edge_of(top, plan.c);
  double sum = 0.0;
  if (top != 0u && plan.bins) {
    const double c16 = plan.c * 16.0, round = exp2.round;
    const double edge_round = fabs(tv * c16) < kLastRounded ? round : 0.0;  // (what is near the largest goes by it)
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float x = (float)line[i][e];
        const double x16 = (double)x * c16, edge = (x16 + edge_round) - edge_round, d = base - edge;
        if (d < (double)(kBins - 1))  // (not for NaN, and not for an infinite top)
          atomicAdd((unsigned long long*)&bin[(uint32_t)__builtin_bit_cast(uint64_t, d + round)],
                    (unsigned long long)bin_word(x16 - edge, bin_exp2));
        else if (x == (float)tv)
          atomicAdd((unsigned long long*)&bin[0], (unsigned long long)bin_word(0.0, bin_exp2));
        else if (x > -INFINITY)  // 2^-39 of the top's weight or less
          sum += weight_called(key_of(x), top, tv, plan.c);
      }
    __syncthreads();
    for (uint32_t i = t; i < kBins; i += kScanThreads) {
      const uint64_t x = bin[i];
      rs.bin[(uint64_t)chunk * kBins + i] = x;
      sum += bin_weight(i, base, tv, plan.c) * (double)(x & kBinMask);
    }
  } else if (top != 0u) {
    const bool finite = tv < INFINITY;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float x = (float)line[i][e];
        // (what has no weight is given 2^-1000 of the top's, which no sum holds;
        // an infinite top's own weight is 1, what lies below has none)
        if (finite)
          sum += exp2_within(fmax(((double)x - tv) * plan.c, -1000.0), exp2);
        else
          sum += x == (float)tv ? 1.0 : 0.0;
      }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  if ((t & 63) == 0) sums[t >> 6] = sum;
  __syncthreads();
  if (t == 0) rs.mass[chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// ---- block-wide sums ------------------------------------------------------------------
// The second kernel's code runs once per launch, from a cold instruction
// cache: what is used often is called, not inlined (a row without filters
// took 35 us with 47 KB of inlined code).

// x moved between lanes by a DPP control; 0 where none comes.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp0(T x) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    int w[W];
  };
  Words a = __builtin_bit_cast(Words, x);
#pragma unroll
  for (int i = 0; i < W; i++) a.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(T, a);
}
template <typename T>
__device__ __forceinline__ T lane_value(T x, int lane) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    int w[W];
  };
  Words a = __builtin_bit_cast(Words, x);
#pragma unroll
  for (int i = 0; i < W; i++) a.w[i] = __builtin_amdgcn_readlane(a.w[i], lane);
  return __builtin_bit_cast(T, a);
}
// Inclusive sum over the wave in lane order.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
  x += dpp0<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += dpp0<0x112, 0xf>(x);
  x += dpp0<0x114, 0xf>(x);
  x += dpp0<0x118, 0xf>(x);
  x += dpp0<0x142, 0xa>(x);  // row_bcast 15, 31
  x += dpp0<0x143, 0xc>(x);
  return x;
}

struct PickShared {
  uint32_t key[kCand];        // gathered values, in index order
  uint32_t index[kCand];
  union {
    struct {
      uint64_t bits[kListed];  // which of the listed groups' values; later the values that are left
      uint16_t list[kListed];  // groups that are read, from the round's first
    };
    struct {
      uint32_t count[kFine];
      uint64_t mass[kFine];
    } fine;
    struct {
      double kept[kMaxChunks];
      double weight[kBins];           // of a unit of a bin's mass
      uint32_t first[kMaxChunks + 1];  // of a chunk's values in key / index
      uint32_t off[kMaxChunks];       // of a chunk's bins from the row's
      uint64_t units[kThreads / 2];
      uint32_t count[kThreads / 2];
    };
  };
  uint32_t group[kCached];
  double factor[kMaxChunks];  // of a chunk's weights; its largest key, its mass
  double mass[kMaxChunks];
  uint32_t top[kMaxChunks];
  uint64_t slots[kWaves];
  uint64_t before;
  uint32_t where[4];
};

// The largest key of group g.
struct Groups {
  const RLH_LDS uint32_t* cached;
  const RLH_GLOBAL uint32_t* all;
  __device__ __forceinline__ uint32_t operator()(uint32_t g) const { return g < kCached ? cached[g] : all[g]; }
};

// Inclusive sum of one value per thread in thread order, and the whole.
template <typename T>
struct Scan {
  T upto, all;
};
template <typename T>
__device__ __noinline__ Scan<T> block_scan(T x, PickShared* sh) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  x = wave_scan(x);
  T* slots = (T*)sh->slots;
  __syncthreads();
  if (lane == 63) slots[wave] = x;
  __syncthreads();
  T v[kWaves], off = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) v[i] = slots[i];
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    off += i < wave ? v[i] : 0;
    sum += v[i];
  }
  return Scan<T>{off + x, sum};
}

// The least key of [lo, hi] for which ok() holds (it does for hi, and for
// all above one for which it does): the wave's lanes try 64 keys at a time.
template <typename F>
__device__ __forceinline__ uint32_t least_key(uint32_t lo, uint32_t hi, F ok) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll 1
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 64 + 1, off = lane * step;
    const uint32_t k = off < hi - lo ? lo + off : hi;
    const uint64_t yes = __ballot(ok(k));
    if (!yes) {
      lo = lane_value(k, 63) + 1;
      continue;
    }
    const int f = __builtin_ctzll(yes);
    hi = lane_value(k, f);
    if (f > 0) lo = lane_value(k, f - 1) + 1;
  }
  return lo;
}

// The border of what is kept: keys above `key`, and of equal ones indices up
// to `index`.
struct Border {
  uint32_t key, index;
};
__device__ __forceinline__ bool kept(const Border& b, uint32_t key, uint32_t index) {
  return key > b.key || (key == b.key && index <= b.index);
}

// f(place, value) for the row's places [from, to) (from: a multiple of 8), by
// `threads` threads of which this is number `mine`; four loads at a time.
template <typename T, typename F>
__device__ __forceinline__ void visit_lines(const Row<T>& row, uint32_t from, uint32_t to, uint32_t mine, uint32_t threads,
                                            F f) {
  constexpr uint32_t V = Row<T>::V;
#pragma unroll 1
  for (uint32_t v0 = from + mine * V; v0 < to; v0 += 4 * threads * V) {
    typename Row<T>::Line line[4];
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) line[q] = row.line(v0 + q * threads * V);
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      const uint32_t v = v0 + q * threads * V;
#pragma unroll
      for (uint32_t e = 0; e < V; e++)
        if (v < to) f(v + e, (float)line[q][e]);
    }
  }
}

// What ends the kept tokens, and what is known of the keys above a range.
struct Goal {
  uint32_t k;        // values (2^32 - 1: no bound)
  double p;          // mass (infinity: no bound)
  uint32_t min_key;  // least key of min_p's weight
  uint32_t top_key;
  double top, c;
};
struct Range {
  uint32_t lo, hi;   // holds the border
  uint32_t above_k;  // values above hi, and their mass
  double above_p;
};

// Narrows the range to one of its 2048 parts by the counts and masses of the
// keys that visit(f) calls f with; false if none of the three bounds ends
// within it.
template <typename F>
__device__ __forceinline__ bool narrow(PickShared& sh, Range& r, const Goal& goal, F visit) {
  const uint32_t t = threadIdx.x, width = r.hi - r.lo;
  const int shift = width < kFine ? 0 : 21 - __builtin_clz(width);
  constexpr uint32_t kPer = kFine / kThreads;
  __syncthreads();
  for (uint32_t i = t; i < kFine; i += kThreads) {
    sh.fine.count[i] = 0;
    sh.fine.mass[i] = 0;
  }
  if (t == 0) sh.where[0] = 0xffffffffu;
  // (2^21 values of at most 2^42 units: below 2^64)
  double unit = 0.0, units = 0.0;  // of a mass; in a weight of one
  if (goal.p < INFINITY) {
    const double most = weight_called(min(r.hi, goal.top_key), goal.top_key, goal.top, goal.c);
    unit = fmax(most, kLeastWeight) * (1.0 / (double)(1ull << kMassBits));
    units = 1.0 / unit;
  }
  __syncthreads();
  visit([&](uint32_t k) {
    if (k < r.lo || k > r.hi) return;
    const uint32_t b = (k - r.lo) >> shift;
    atomicAdd(&sh.fine.count[b], 1u);
    if (goal.p < INFINITY)
      atomicAdd((unsigned long long*)&sh.fine.mass[b],
                (unsigned long long)(weight_called(k, goal.top_key, goal.top, goal.c) * units + 0.5));
  });
  __syncthreads();
  // each thread's parts, from the top
  uint32_t ck = 0;
  uint64_t cp = 0;
  for (uint32_t j = 0; j < kPer; j++) {
    ck += sh.fine.count[kFine - 1 - t * kPer - j];
    cp += sh.fine.mass[kFine - 1 - t * kPer - j];
  }
  uint32_t upto_k = block_scan<uint32_t>(ck, &sh).upto - ck;
  uint64_t upto_p = goal.p < INFINITY ? block_scan<uint64_t>(cp, &sh).upto - cp : 0;
  uint32_t mine = 0xffffffffu;
  for (uint32_t j = 0; j < kPer; j++) {
    const uint32_t b = kFine - 1 - t * kPer - j;
    if (b > width >> shift) continue;
    const uint64_t part = sh.fine.mass[b];
    const uint32_t cnt = sh.fine.count[b];
    if ((goal.k != 0xffffffffu && r.above_k + upto_k + cnt >= goal.k) ||
        r.above_p + (double)(upto_p + part) * unit >= goal.p ||
        r.lo + (b << shift) < goal.min_key) {
      mine = kFine - 1 - b;
      break;
    }
    upto_k += cnt;
    upto_p += part;
  }
  const uint64_t ends = __ballot(mine != 0xffffffffu);
  if (ends && (int)(t & 63) == __builtin_ctzll(ends)) atomicMin(&sh.where[0], mine);
  __syncthreads();
  const uint32_t found = sh.where[0];
  if (found == 0xffffffffu) return false;
  const uint32_t b = kFine - 1 - found;
  if (found == mine) {
    sh.where[1] = upto_k;
    sh.before = upto_p;
  }
  __syncthreads();
  r.above_k += sh.where[1];
  r.above_p += (double)sh.before * unit;
  r.lo += b << shift;
  r.hi = r.lo + min(r.hi - r.lo, (1u << shift) - 1);
  __syncthreads();
  return true;
}

// How many of n equal values (key lo of a range that is one key) are kept.
__device__ __forceinline__ uint32_t kept_equal(const Range& r, const Goal& goal, uint32_t n) {
  uint32_t m = n;
  if (goal.k != 0xffffffffu) m = min(m, goal.k > r.above_k ? goal.k - r.above_k : 0u);
  if (goal.p < INFINITY) {
    const double w = weight_called(r.lo, goal.top_key, goal.top, goal.c);
    const double d = w > 0.0 ? ceil((goal.p - r.above_p) / w) : 0.0;
    if (d < (double)m) m = d > 0.0 ? (uint32_t)d : 0u;
  }
  if (r.lo < goal.min_key) m = 0;
  if (r.lo == goal.top_key) m = max(m, 1u);
  return m;
}

// Every value with key in [lo, hi] into sh.key / sh.index, in index order;
// false when there are more than kCand. Reads the groups that reach lo.
template <typename T>
__device__ __forceinline__ bool gather(PickShared& sh, const Row<T>& row, const Groups& group, uint32_t groups,
                                       uint32_t lo, uint32_t hi, uint32_t* count) {
  constexpr uint32_t V = Row<T>::V;
  constexpr uint32_t kLanes = kGroup / V;  // of a group; a wave takes V groups
  constexpr uint64_t kEach = ~0ull / ((1ull << kLanes) - 1);  // a lane's bits
  // the range as values (the keys of -infinity and NaN are below lo)
  const float least = value_of(max(lo, kLeastKey)), most = value_of(min(hi, kMostKey));
  const uint32_t outside = row.lines() + V;  // of the row (a place that no line has)
  const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
  uint32_t found = 0;
  // rounds of neighbouring groups, eight per thread if the list holds those
  // that reach lo, else five
  uint32_t per = 8;
#pragma unroll 1
  for (uint32_t g0 = 0; g0 < groups;) {
    const uint32_t first = g0 + t * per;
    uint32_t yes = 0;
    for (uint32_t j = 0; j < per; j++) yes |= (first + j < groups && group(first + j) >= lo ? 1u : 0u) << j;
    const Scan<uint32_t> places = block_scan<uint32_t>((uint32_t)__popc(yes), &sh);
    uint32_t at = places.upto - (uint32_t)__popc(yes);
    const uint32_t listed = places.all;
    if (listed > kListed) {  // (not with five: those are kListed at most)
      per = kListed / kThreads;
      continue;
    }
    for (; yes; yes &= yes - 1, at++) sh.list[at] = (uint16_t)(first - g0 + (uint32_t)__builtin_ctz(yes));
    __syncthreads();
    // which values of each group, 16 groups' loads at a time. A wave's V
    // groups leave V words: word e has value e of each lane
    constexpr uint32_t kBatch = 16;
#pragma unroll 1
    for (uint32_t i0 = wave * V; i0 < listed; i0 += kBatch * kWaves * V) {
      typename Row<T>::Line line[kBatch];
#pragma unroll
      for (uint32_t q = 0; q < kBatch; q++) {
        if (i0 + q * kWaves * V >= listed) break;
        const uint32_t i = i0 + q * kWaves * V + lane / kLanes;
        line[q] = row.line(i < listed ? (g0 + sh.list[i]) * kGroup + lane % kLanes * V : outside);
      }
#pragma unroll
      for (uint32_t q = 0; q < kBatch; q++) {
        if (i0 + q * kWaves * V >= listed) break;
        uint64_t word = 0;
#pragma unroll
        for (uint32_t e = 0; e < V; e++) {
          const float x = (float)line[q][e];
          const uint64_t in = __ballot(x >= least && x <= most);
          word = lane == e ? in : word;
        }
        const uint32_t i = i0 + q * kWaves * V + lane;
        if (lane < V) sh.bits[i] = word;
      }
    }
    __syncthreads();
    // the places of their values: five neighbours per thread
    auto values_of = [&](uint32_t i) {  // bit e * kLanes + lane
      uint64_t x = 0;
#pragma unroll
      for (uint32_t e = 0; e < V; e++)
        x |= (sh.bits[i / V * V + e] >> (i % V * kLanes) & ((1ull << kLanes) - 1)) << (e * kLanes);
      return x;
    };
    uint32_t n = 0;
    uint64_t own[kListed / kThreads];
    const uint32_t l0 = t * (kListed / kThreads);
#pragma unroll
    for (uint32_t j = 0; j < kListed / kThreads; j++) {
      own[j] = l0 + j < listed ? values_of(l0 + j) : 0ull;
      n += (uint32_t)__popcll(own[j]);
    }
    const Scan<uint32_t> values = block_scan<uint32_t>(n, &sh);
    uint32_t to = found + values.upto - n;
#pragma unroll
    for (uint32_t j = 0; j < kListed / kThreads; j++) {
      uint64_t left = own[j];
#pragma unroll 1
      while (left) {  // the lanes in order, of each its values
        uint64_t any = left;
#pragma unroll
        for (uint32_t e = kLanes; e < 64; e <<= 1) any |= any >> e;
        const uint32_t l = (uint32_t)__builtin_ctzll(any);
        uint64_t of_lane = left >> l & kEach;
        left &= ~(kEach << l);
        for (; of_lane; of_lane &= of_lane - 1, to++)
          if (to < kCand) sh.index[to] = (g0 + sh.list[l0 + j]) * kGroup + l * V + (uint32_t)__builtin_ctzll(of_lane) / kLanes;
      }
    }
    g0 += per * kThreads;
    found += values.all;
    __syncthreads();
    if (found > kCand) return false;
  }
  for (uint32_t i = t; i < found; i += kThreads) sh.key[i] = row.key(sh.index[i]);
  __syncthreads();
  *count = found;
  return true;
}

// The index of the nth (from 1) value that equals key.
template <typename T>
__device__ __noinline__ uint32_t nth_equal(PickShared* sh, const Row<T> row, uint32_t key, uint32_t nth) {
  uint32_t seen = 0;
  for (uint32_t v0 = 0; v0 < row.lines() && seen < nth; v0 += kThreads) {
    const uint32_t v = v0 + threadIdx.x, yes = v < row.lines() && row.key(v) == key ? 1u : 0u;
    const Scan<uint32_t> c = block_scan<uint32_t>(yes, sh);
    if (yes && seen + c.upto == nth) sh->where[2] = v;
    seen += c.all;
  }
  __syncthreads();
  const uint32_t v = sh->where[2];
  __syncthreads();
  return v;
}

// The border within a range: gathers it (after narrowing over the whole row
// while it holds too many), narrows the gathered list, sorts what is left.
// *gathered: values in sh.key / sh.index if they are the whole of the first
// range, else 2^32 - 1.
template <typename T>
__device__ __noinline__ Border find_border(PickShared* shp, const Row<T> row, const Groups group, uint32_t groups,
                                           Range r, const Goal goal, uint32_t* gathered) {
  PickShared& sh = *shp;
  const uint32_t t = threadIdx.x, lane = t & 63;
  uint32_t m = 0;
  bool whole = true;
#pragma unroll 1
  while (!gather(sh, row, group, groups, r.lo, r.hi, &m)) {
    whole = false;
    if (r.lo == r.hi) {
      // more equal values than the list holds
      uint32_t part = 0;
      for (uint32_t v = t; v < row.lines(); v += kThreads) part += row.key(v) == r.lo ? 1u : 0u;
      const uint32_t n = kept_equal(r, goal, block_scan<uint32_t>(part, shp).all);
      *gathered = 0xffffffffu;
      return n ? Border{r.lo, nth_equal(shp, row, r.lo, n)} : Border{r.lo + 1, 0xffffffffu};
    }
    const float least = value_of(max(r.lo, kLeastKey)), most = value_of(min(r.hi, kMostKey));
    if (!narrow(sh, r, goal, [&](auto f) {
          visit_lines(row, 0u, row.lines(), t, (uint32_t)kThreads, [&](uint32_t, float x) {
            if (x >= least && x <= most) f(key_of(x));
          });
        })) {
      *gathered = 0xffffffffu;
      return Border{r.lo, 0xffffffffu};
    }
  }
  *gathered = whole ? m : 0xffffffffu;
  if (m > 64) {
    while (r.lo != r.hi) {
      if (!narrow(sh, r, goal, [&](auto f) {
            for (uint32_t i = t; i < m; i += kThreads) f(sh.key[i]);
          })) return Border{r.lo, 0xffffffffu};
      uint32_t in = 0;
      for (uint32_t i = t; i < m; i += kThreads) in += sh.key[i] >= r.lo && sh.key[i] <= r.hi ? 1u : 0u;
      if (block_scan<uint32_t>(in, shp).all <= 64) break;
    }
  }
  // what is left, in index order: four neighbours per thread
  uint32_t in = 0;
  const uint32_t i0 = t * (kCand / kThreads);
  for (uint32_t j = 0; j < kCand / kThreads; j++)
    in |= (i0 + j < m && sh.key[i0 + j] >= r.lo && sh.key[i0 + j] <= r.hi ? 1u : 0u) << j;
  const Scan<uint32_t> places = block_scan<uint32_t>((uint32_t)__popc(in), shp);
  const uint32_t left = places.all;
  uint32_t at = places.upto - (uint32_t)__popc(in);
  for (; in; in &= in - 1, at++) {
    const uint32_t i = i0 + (uint32_t)__builtin_ctz(in);
    sh.bits[at] = (uint64_t)sh.key[i] << 32 | (uint32_t)~sh.index[i];
  }
  __syncthreads();
  if (left > 64) {  // equal values
    const uint32_t n = kept_equal(r, goal, left);
    return n ? Border{r.lo, ~(uint32_t)sh.bits[n - 1]} : Border{r.lo + 1, 0xffffffffu};
  }
  if (t < 64) {
    // each by the number of larger ones (no two are equal)
    const uint64_t own = lane < left ? sh.bits[lane] : 0ull;
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t i = 0; i < left; i++) rank += sh.bits[i] > own ? 1u : 0u;
    if (lane < left) sh.bits[64 + rank] = own;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint64_t k = lane < left ? sh.bits[64 + lane] : 0ull;
    const uint32_t key = (uint32_t)(k >> 32);
    const double w = lane < left ? weight_called(key, goal.top_key, goal.top, goal.c) : 0.0;
    const double before = r.above_p + (wave_scan(w) - w);
    const bool keep = lane < left && ((goal.k == 0xffffffffu || r.above_k + lane < goal.k) && before < goal.p &&
                                      key >= goal.min_key);
    uint64_t dropped = __ballot(!keep);
    if (left && r.above_k == 0 && lane_value((uint32_t)(k >> 32), 0) == goal.top_key) dropped &= ~1ull;  // the row's first
    const uint32_t n = dropped ? (uint32_t)__builtin_ctzll(dropped) : 64u;
    const uint64_t last = lane_value(k, n ? (int)n - 1 : 0);
    if (t == 0) {
      sh.where[0] = n ? (uint32_t)(last >> 32) : r.hi + 1;
      sh.where[1] = n ? ~(uint32_t)last : 0xffffffffu;
    }
  }
  __syncthreads();
  const Border b{sh.where[0], sh.where[1]};
  __syncthreads();
  return b;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_pick(const T* logits, uint32_t n, uint64_t stride,
                                                          const rlh_row_sampling* options, const float* us,
                                                          uint32_t* tokens, Space space) {
  __shared__ PickShared sh;
  const uint32_t t = threadIdx.x, r = blockIdx.x, lane = t & 63, wave = t >> 6;
  const rlh_row_sampling o = options[r];
  const float u = us[r];
  const RowSpace rs = space.row(r);
  const Row<T> row(logits, stride, n, r);
  const uint32_t chunks = (row.lines() + kChunk - 1) / kChunk, groups = (row.lines() + kGroup - 1) / kGroup;
  // what the first launch left, all loads at once: a chain of loads that wait
  // for each other costs most of the time here
  uint32_t top_key = 0;
  uint32_t g[kCached / kThreads];
#pragma unroll
  for (uint32_t j = 0; j < kCached / kThreads; j++) g[j] = j * kThreads + t < groups ? rs.group[j * kThreads + t] : 0u;
  for (uint32_t i = t; i < chunks; i += kThreads) {
    const uint32_t k = rs.top[i];
    sh.top[i] = k;
    sh.mass[i] = rs.mass[i];  // (not written, and not used, where the plan asks for no masses)
    top_key = max(top_key, k);
  }
#pragma unroll
  for (uint32_t j = 0; j < kCached / kThreads; j++) sh.group[j * kThreads + t] = g[j];
  const Groups group{(const RLH_LDS uint32_t*)sh.group, (const RLH_GLOBAL uint32_t*)rs.group};
  const RowPlan plan = row_plan(o, n);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top_key = max(top_key, (uint32_t)__shfl_xor((int)top_key, d));
  uint32_t* tops = (uint32_t*)sh.slots;
  if (lane == 0) tops[wave] = top_key;
  if (t == 0) sh.where[0] = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) top_key = max(top_key, tops[i]);
  if (top_key == 0u) {
    if (t == 0) tokens[r] = 0;
    return;
  }
  if (plan.greedy) {
    // the first group that holds it, the first of its values
    for (uint32_t i = t; i < groups; i += kThreads)
      if (group(i) == top_key) {
        atomicMin(&sh.where[0], i);
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
  const double top = (double)value_of(top_key), c = plan.c;
  // masses of chunks are relative to their own largest weight
  Goal goal{plan.by_k ? o.top_k : 0xffffffffu, INFINITY, 0u, top_key, top, c};
  if (plan.mass) {
    double part = 0.0;
    for (uint32_t i = t; i < chunks; i += kThreads) {
      const double f = weight_called(sh.top[i], top_key, top, c);
      sh.factor[i] = f;
      part += f * sh.mass[i];
    }
    const double sum = block_scan<double>(part, &sh).all;
    if (plan.by_p) goal.p = (double)o.top_p * sum;
  }
  if (plan.min_p > 0.0) {
    const uint32_t lo = least_key(1, top_key, [&](uint32_t k) { return weight_called(k, top_key, top, c) >= plan.min_p; });
    goal.min_key = plan.min_p > 1.0 ? top_key + 1 : lo;
  }
  const double uu = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
  const double base = edge_of(top_key, c);

  Border border{0u, 0xffffffffu};  // everything
  uint32_t border_bin = kBins, m = 0xffffffffu;
  if (plan.list) {
    // a key that at least k groups reach, to a 2048th of the maxima's span
    uint32_t least = 0xffffffffu;
    for (uint32_t i = t; i < groups; i += kThreads) least = min(least, group(i) ? group(i) : 0xffffffffu);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d));
    __syncthreads();
    if (lane == 0) tops[wave] = least;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; i++) least = min(least, tops[i]);
    Range range{least, top_key, 0u, 0.0};
    const Goal by_count{o.top_k, INFINITY, 0u, top_key, top, c};
    const bool enough = narrow(sh, range, by_count, [&](auto f) {
      for (uint32_t i = t; i < groups; i += kThreads) f(group(i));
    });
    range = Range{enough ? range.lo : 1u, 0xffffffffu, 0u, 0.0};
    border = find_border(&sh, row, group, groups, range, goal, &m);
  } else if (plan.bins) {
    // the row's histogram, 16 powers of two at a time until one of the three
    // bounds ends: a bin per thread, half of the chunks for each half of the
    // block. (One block reads 31 GB/s whatever it asks for at once, so it asks
    // for little: all 640 bins of 38 chunks took 10 us.) The row's bins lie
    // off[chunk] before the chunk's.
    for (uint32_t i = t; i < chunks; i += kThreads) sh.off[i] = sh.top[i] ? bin_of(sh.top[i], top_key, base, c) : kBins;
    if (t == 0) sh.where[0] = 0xffffffffu;
    __syncthreads();
    constexpr uint32_t kHalf = kThreads / 2;
    const uint32_t min_bin = goal.min_key == 0u ? kBins : bin_of(min(goal.min_key, top_key), top_key, base, c);
    uint32_t above_k = 0;
    double above_p = 0.0;
#pragma unroll 1
    for (uint32_t b0 = 0; b0 < kBins - 1; b0 += kHalf) {
      const uint32_t b = b0 + t % kHalf;
      uint32_t cnt = 0;
      uint64_t units = 0;  // (2^21 values of up to 2^38.1: below 2^60)
#pragma unroll 8
      for (uint32_t ch = t / kHalf; ch < chunks; ch += 2) {
        // (bin 0 is read and not used where the chunk has none)
        const uint32_t off = sh.off[ch];
        const bool in = b >= off && b < kBins - 1;
        const uint64_t x = rs.bin[(uint64_t)ch * kBins + (in ? b - off : 0u)];
        cnt += in ? (uint32_t)(x >> kBinShift) : 0u;
        units += in ? x & kBinMask : 0ull;
      }
      if (t >= kHalf) {
        sh.units[t - kHalf] = units;
        sh.count[t - kHalf] = cnt;
        cnt = 0;
        units = 0;
      }
      __syncthreads();
      if (t < kHalf) {
        units += sh.units[t];
        cnt += sh.count[t];
      }
      const double mass = t < kHalf ? (double)units * bin_weight(b, base, top, c) : 0.0;
      const Scan<uint32_t> sum_k = block_scan<uint32_t>(cnt, &sh);
      const Scan<double> sum_p = block_scan<double>(mass, &sh);
      // the first bin at which one of the three ends
      const bool ends = t < kHalf && b < kBins - 1 &&
                        ((plan.by_k && above_k + sum_k.upto >= o.top_k) || (plan.by_p && above_p + sum_p.upto >= goal.p) || b >= min_bin);
      const uint64_t any = __ballot(ends);
      if (any && (int)lane == __builtin_ctzll(any)) atomicMin(&sh.where[0], b);
      __syncthreads();
      border_bin = sh.where[0];
      if (t < kHalf && b == border_bin) {
        sh.where[1] = above_k + sum_k.upto - cnt;
        sh.before = __builtin_bit_cast(uint64_t, above_p + (sum_p.upto - mass));
      }
      if (border_bin != 0xffffffffu) break;
      above_k += sum_k.all;
      above_p += sum_p.all;
    }
    // the bin's keys: bins fall as keys rise. Where no bound ends within the
    // bins, one may among what lies below them and has weight
    const bool deep = border_bin == 0xffffffffu;
    if (deep) border_bin = kBins - 1;
    auto from_bin = [&](uint32_t b) { return least_key(1, top_key, [&](uint32_t k) { return bin_of(k, top_key, base, c) <= b; }); };
    // the first half of the waves looks for the bin's end, the others for the next one's
    const bool low = wave < kWaves / 2;
    uint32_t edge = top_key + 1;
    if (low && deep)
      edge = least_key(1, top_key, [&](uint32_t k) { return weight_called(k, top_key, top, c) >= kLeastWeight; });
    else if (low || border_bin > 0)
      edge = from_bin(low ? border_bin : border_bin - 1);
    if (lane == 0 && wave % (kWaves / 2) == 0) sh.where[low ? 2 : 3] = edge;
    __syncthreads();
    const uint32_t lo = sh.where[2], hi = sh.where[3] - 1;
    const Range range{lo, hi, deep ? above_k : sh.where[1], deep ? above_p : __builtin_bit_cast(double, sh.before)};
    border = find_border(&sh, row, group, groups, range, goal, &m);
  }
  __syncthreads();
  uint32_t per = 0, ch = 0;  // neighbours per thread of the list; or the draw's chunk
  double before = 0.0, draw = 0.0, least_weight = kLeastWeight;
  const bool at_end = !(uu < 1.0);  // nothing exceeds the draw: the last that has weight
  const bool from_list = plan.list && m != 0xffffffffu;
  if (from_list) {
    per = (m + kThreads - 1) / kThreads;
  } else {
    // the draw over the chunks' kept masses
    if (border.key == 0u) {
      for (uint32_t q = t; q < chunks; q += kThreads) sh.kept[q] = sh.top[q] ? sh.factor[q] * sh.mass[q] : 0.0;
    } else {
      const float least = value_of(max(border.key, kLeastKey));
      const bool by_bins = border_bin < kBins && m != 0xffffffffu;
      if (by_bins) {
        // where each chunk's values begin in the list
        for (uint32_t i = t; i <= m; i += kThreads) {
          const uint32_t upto = i < m ? sh.index[i] / kChunk : chunks;
          for (uint32_t q = i ? sh.index[i - 1] / kChunk + 1 : 0u; q <= upto; q++) sh.first[q] = i;
        }
        for (uint32_t i = t; i < kBins; i += kThreads) sh.weight[i] = bin_weight(i, base, top, c);
        for (uint32_t i = t; i < chunks; i += kThreads) sh.off[i] = sh.top[i] ? bin_of(sh.top[i], top_key, base, c) : kBins;
        __syncthreads();
      }
#pragma unroll 1
      for (uint32_t q = wave; q < chunks; q += kWaves) {
        const uint32_t ck = sh.top[q];
        double s = 0.0;
        if (ck != 0u && ck >= border.key) {
          if (by_bins) {
            // the bins above the border's, and what is kept of that one
            const uint32_t off = sh.off[q];
#pragma unroll 1
            for (uint32_t i0 = 0; off + i0 < border_bin; i0 += kBins / 2) {
              uint64_t x[kBins / 128];
#pragma unroll
              for (uint32_t j = 0; j < kBins / 128; j++) x[j] = rs.bin[(uint64_t)q * kBins + i0 + j * 64 + lane];
#pragma unroll
              for (uint32_t j = 0; j < kBins / 128; j++) {
                const uint32_t b = off + i0 + j * 64 + lane;
                if (b < border_bin) s += sh.weight[b] * (double)(x[j] & kBinMask);
              }
            }
            for (uint32_t i = sh.first[q] + lane; i < sh.first[q + 1]; i += 64)
              if (kept(border, sh.key[i], sh.index[i])) s += weight_called(sh.key[i], top_key, top, c);
          } else {
            visit_lines(row, q * kChunk, (q + 1) * kChunk, lane, 64u, [&](uint32_t v, float x) {
              if (!(x >= least)) return;
              const uint32_t k = key_of(x);
              if (kept(border, k, v)) s += weight_called(k, top_key, top, c);
            });
          }
        }
        s = wave_scan(s);
        if (lane == 63) sh.kept[q] = s;
      }
    }
    if (t == 0) {
      sh.where[0] = 0xffffffffu;
      sh.where[1] = 0;
    }
    __syncthreads();
    // two chunks per thread (there are at most 513)
    const double a = 2 * t < chunks ? sh.kept[2 * t] : 0.0, b = 2 * t + 1 < chunks ? sh.kept[2 * t + 1] : 0.0;
    const Scan<double> sums = block_scan<double>(a + b, &sh);
    const double at = sums.upto - (a + b);
    draw = uu * sums.all;
    if (!at_end) {
      if (a > 0.0 && at + a > draw) atomicMin(&sh.where[0], 2 * t);
      if (b > 0.0 && at + a + b > draw) atomicMin(&sh.where[0], 2 * t + 1);
    }
    __syncthreads();
    ch = sh.where[0];
    if (ch == 0xffffffffu) {
      // the last chunk that has a kept weight of kLeastWeight: its largest is
      // kept if any is (the row's largest always: there is one)
      if (b > 0.0 && weight_called(sh.top[2 * t + 1], top_key, top, c) >= kLeastWeight)
        atomicMax(&sh.where[1], 2 * t + 1);
      else if (a > 0.0 && weight_called(sh.top[2 * t], top_key, top, c) >= kLeastWeight)
        atomicMax(&sh.where[1], 2 * t);
      __syncthreads();
      ch = sh.where[1];
    } else {
      // (found by sums of another order than those below: the draw may lie past
      // the chunk's end by their last bits, and the chunk may have little weight)
      least_weight *= fmin(1.0, sh.kept[ch]);
    }
    if (ch / 2 == t) sh.before = __builtin_bit_cast(uint64_t, ch % 2 ? at + a : at);
    __syncthreads();
    before = __builtin_bit_cast(double, sh.before);
  }
  if (t == 0) {
    sh.where[2] = 0xffffffffu;
    sh.where[3] = 0;
  }
  // the draw over neighbouring values per thread, so that sums in thread order
  // are in index order
  constexpr uint32_t kPer = kChunk / kThreads, V = Row<T>::V;
  double w[kPer], s = 0.0;
  uint32_t at[kPer], k[kPer];
  if (from_list) {
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) {
      const uint32_t i = t * per + j;
      const bool in = j < per && i < m;
      at[j] = in ? sh.index[i] : 0u;
      k[j] = in ? sh.key[i] : 0u;
    }
  } else {
    typename Row<T>::Line line[kPer / V];
#pragma unroll
    for (uint32_t j = 0; j < kPer / V; j++) line[j] = row.line(ch * kChunk + t * kPer + j * V);
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) k[j] = key_of((float)line[j / V][j % V]);
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) at[j] = ch * kChunk + t * kPer + j;
  }
#pragma unroll
  for (uint32_t j = 0; j < kPer; j++) {
    w[j] = k[j] != 0u && kept(border, k[j], at[j]) ? weight_called(k[j], top_key, top, c) : 0.0;
    s += w[j];
  }
  const Scan<double> sums = block_scan<double>(s, &sh);
  double run = sums.upto - s + before;
  if (from_list) draw = uu * sums.all;
  if (at_end) draw = INFINITY;
  uint32_t hit = 0xffffffffu, last = 0xffffffffu;
#pragma unroll
  for (uint32_t j = 0; j < kPer; j++) {
    run += w[j];
    if (hit == 0xffffffffu && w[j] > 0.0 && run > draw) hit = at[j];
    if (w[j] >= least_weight) last = at[j];
  }
  // one lane of a wave speaks for it: the sums rise and the indices with them
  const uint64_t hits = __ballot(hit != 0xffffffffu), lasts = __ballot(last != 0xffffffffu);
  if (hits && (int)lane == __builtin_ctzll(hits)) atomicMin(&sh.where[2], hit);
  if (lasts && (int)lane == 63 - __builtin_clzll(lasts)) atomicMax(&sh.where[3], last);
  __syncthreads();
  // (none past the draw: u at its upper end, or sums that differ in their last
  // bits; a token of least_weight there is)
  if (t == 0) tokens[r] = (sh.where[2] != 0xffffffffu ? sh.where[2] : sh.where[3]) - row.shift;
}

Space sample_space(void* base, uint64_t n) {
  Space s;
  s.base = (uint8_t*)base;
  // a row may begin up to 7 values into its first line
  s.chunks = (uint32_t)((n + 7 + kChunk - 1) / kChunk);
  s.groups = (uint32_t)((n + 7 + kGroup - 1) / kGroup);
  s.row_bytes = ((uint64_t)s.chunks * (kBins * 8 + 12) + (uint64_t)s.groups * 4 + 255) / 256 * 256;
  return s;
}

template <typename T>
int launch_sample(const void* logits, uint64_t n_rows, uint64_t n, uint64_t stride, const rlh_row_sampling* options,
                  const float* u, uint32_t* tokens, const Space& space, hipStream_t s) {
  const dim3 chunks(space.chunks * (uint32_t)n_rows), rows((uint32_t)n_rows);
  const T* x = (const T*)logits;
  RLH_TRY(enqueue("rlh_sample_rows", k_sample_scan<T>, chunks, kScanThreads, 0, s, x, (uint32_t)n, stride, options, space));
  return enqueue("rlh_sample_rows", k_sample_pick<T>, rows, kThreads, 0, s, x, (uint32_t)n, stride, options, u, tokens, space);
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
    return serve_error(RLH_EUNSUP, "more than 2^21 rows, or 2^35 logits");
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
  const uint64_t span = row_bytes_span(n_rows, stride, n, size);
  if (overlap(workspace, need, logits, span) || overlap(workspace, need, options, n_rows * sizeof(*options)) ||
      overlap(workspace, need, u, n_rows * 4) || overlap(workspace, need, tokens, n_rows * 4) ||
      overlap(tokens, n_rows * 4, logits, span) || overlap(tokens, n_rows * 4, options, n_rows * sizeof(*options)) ||
      overlap(tokens, n_rows * 4, u, n_rows * 4))
    return serve_error(RLH_EINVAL, "workspace or tokens overlap another argument");
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("logits", logits));
  RLH_TRY(dev("options", options));
  RLH_TRY(dev("u", u));
  RLH_TRY(dev("tokens", tokens));
  if (need) RLH_TRY(dev("workspace", workspace));
  hipStream_t s = (hipStream_t)stream;
  const Space space = sample_space(workspace, n);
  if (type == RLH_TYPE_F32) return launch_sample<float>(logits, n_rows, n, stride, options, u, tokens, space, s);
  if (type == RLH_TYPE_F16) return launch_sample<_Float16>(logits, n_rows, n, stride, options, u, tokens, space, s);
  return launch_sample<__bf16>(logits, n_rows, n, stride, options, u, tokens, space, s);
}

}  // extern "C"
