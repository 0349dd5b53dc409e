// sample_rows.hip — one token per row of logits: temperature, top-k, top-p
// and min-p from given random numbers.
#include <math.h>

#include "paged_device.h"
#include "serve_check.h"

namespace rlh {
namespace {

// Masses are whole multiples of 2^-42 of the largest weight: their sums do
// not depend on an order, and 2^21 of them fit 64 bits.
constexpr int kMassBits = 42;
constexpr uint64_t kMaxRow = 1ull << 21;
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kBins = 2048;

// Ascending as the values are; NaN (either sign) and -infinity give 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);  // -0 equals 0
  if (!(x > -INFINITY)) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp((x - top) / temperature) in 64 bits; 1 at the top itself (so infinite
// tops share the mass), 0 for what has none.
__device__ __forceinline__ double weight_of(uint32_t key, float top, float heat) {
  if (key == 0u) return 0.0;
  const float x = value_of(key);
  if (x == top) return 1.0;
  const double e = exp(((double)x - (double)top) / (double)heat);
  return e == e ? e : 0.0;
}
__device__ __forceinline__ uint64_t mass_of(double w) { return (uint64_t)(w * (double)(1ull << kMassBits) + 0.5); }

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* slots) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = 0;
  for (int i = 0; i < kWaves; i++) r += slots[i];
  return r;
}

// The bin (from the top) at which the running sum over bins first reaches
// `goal`; *before receives the sum above it. kBins bins, two per thread.
template <typename T, typename F>
__device__ __forceinline__ uint32_t find_bin(const T* bins, F reached, T* before, T* slots, uint32_t* where) {
  const int t = threadIdx.x;
  const uint32_t hi = kBins - 1 - 2 * t, lo = hi - 1;
  const T a = bins[hi], b = bins[lo];
  T inc = a + b;
  for (int m = 1; m < 64; m <<= 1) {
    const T o = __shfl_up(inc, m);
    if ((t & 63) >= m) inc += o;
  }
  __syncthreads();
  if ((t & 63) == 63) slots[t >> 6] = inc;
  if (t == 0) *where = 0;
  __syncthreads();
  T off = 0;
  for (int i = 0; i < (t >> 6); i++) off += slots[i];
  const T pre = off + inc - a - b;
  __syncthreads();
  if (!reached(pre) && reached(pre + a)) {
    *where = hi;
    slots[0] = pre;
  } else if (!reached(pre + a) && reached(pre + a + b)) {
    *where = lo;
    slots[0] = pre + a;
  }
  __syncthreads();
  *before = slots[0];
  const uint32_t r = *where;
  __syncthreads();
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_row(const T* logits, uint64_t n64, uint64_t stride,
                                                         const rlh_row_sampling* options, const float* us,
                                                         uint32_t* tokens) {
  __shared__ uint32_t cbin[kBins];
  __shared__ uint64_t mbin[kBins];
  __shared__ uint64_t slots[kWaves];
  __shared__ uint32_t slots32[kWaves];
  __shared__ uint32_t where;
  const uint32_t n = (uint32_t)n64, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const T* x = logits + (size_t)blockIdx.x * stride;
  const rlh_row_sampling o = options[blockIdx.x];
  // the first of the order: largest key, lowest index
  uint64_t best = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    const uint64_t c = ((uint64_t)key_of((float)x[i]) << 32) | (uint32_t)~i;
    best = c > best ? c : best;
  }
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t c = __shfl_xor((unsigned long long)best, m);
    best = c > best ? c : best;
  }
  if (lane == 0) slots[wave] = best;
  __syncthreads();
  for (int i = 0; i < kWaves; i++) best = slots[i] > best ? slots[i] : best;
  __syncthreads();
  const uint32_t top_key = (uint32_t)(best >> 32), first = ~(uint32_t)best;
  const bool greedy = !(o.temperature > 0.0f);
  if (top_key == 0u || greedy) {
    if (t == 0) tokens[blockIdx.x] = top_key == 0u ? 0u : first;
    return;
  }
  const float top = value_of(top_key), heat = o.temperature;
  const bool by_k = o.top_k > 0 && o.top_k < n;
  const bool by_p = o.top_p > 0.0f && o.top_p < 1.0f;
  const double min_p = o.min_p > 0.0f ? (double)o.min_p : 0.0;
  uint64_t part = 0;
  if (by_p)
    for (uint32_t i = t; i < n; i += kThreads) part += mass_of(weight_of(key_of((float)x[i]), top, heat));
  const double goal_p = by_p ? (double)o.top_p * (double)block_sum(part, slots) : 0.0;
  const uint32_t goal_k = o.top_k;
  // threshold keys by radix descent: 11, 11 and 10 bits
  uint32_t key_k = 0, key_p = 0, above_k = 0;
  uint64_t above_p = 0;
  for (int r = 0; r < 3; r++) {
    if (!by_k && !by_p) break;
    const int shift = r == 0 ? 21 : r == 1 ? 10 : 0;
    const uint32_t mask = r == 0 ? 0u : r == 1 ? 0xffe00000u : 0xfffffc00u;
    for (uint32_t i = t; i < kBins; i += kThreads) {
      cbin[i] = 0;
      mbin[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = t; i < n; i += kThreads) {
      const uint32_t k = key_of((float)x[i]);
      if (k == 0u) continue;
      const uint32_t b = (k >> shift) & (r == 2 ? 1023u : 2047u);
      if (by_k && ((k ^ key_k) & mask) == 0) atomicAdd(&cbin[b], 1u);
      if (by_p && ((k ^ key_p) & mask) == 0)
        atomicAdd((unsigned long long*)&mbin[b], (unsigned long long)mass_of(weight_of(k, top, heat)));
    }
    __syncthreads();
    if (by_k) {
      uint32_t before;
      const uint32_t base = above_k;
      const uint32_t b = find_bin<uint32_t>(cbin, [&](uint32_t v) { return base + v >= goal_k; }, &before, slots32, &where);
      key_k |= b << shift;
      above_k += before;
    }
    if (by_p) {
      uint64_t before;
      const uint64_t base = above_p;
      const uint32_t b =
          find_bin<uint64_t>(mbin, [&](uint64_t v) { return (double)(base + v) >= goal_p && base + v > 0; }, &before, slots, &where);
      key_p |= b << shift;
      above_p += before;
    }
    __syncthreads();
  }
  // kept: keys above `key`, and the first `ties` of those equal to it
  uint32_t key = 1, ties = 0xffffffffu;
  if (by_k && key_k != 0u) {  // (0: fewer than top_k values have a key)
    key = key_k;
    ties = goal_k - above_k;
  }
  if (by_p) {
    const uint64_t w = mass_of(weight_of(key_p, top, heat));
    uint32_t r = 1;
    if (w > 0) {
      const double d = (goal_p - (double)above_p) / (double)w;
      r = d > 1.0 ? (uint32_t)fmin(d, 2097152.0) : 1u;
      while (r > 1 && (double)(above_p + (uint64_t)(r - 1) * w) >= goal_p) r--;
      while ((double)(above_p + (uint64_t)r * w) < goal_p && r < n) r++;
    }
    if (key_p > key || (key_p == key && r < ties)) {
      key = key_p;
      ties = r;
    }
  }
  // kept mass of each wave's run of indices
  const uint32_t seg = ((n + kWaves - 1) / kWaves + 63) / 64 * 64;
  const uint32_t i0 = wave * seg, i1 = min(n, i0 + seg);
  uint64_t mass = 0;
  uint32_t eq = 0;
  auto kept_mass = [&](uint32_t k) -> uint64_t {
    const double w = weight_of(k, top, heat);
    return k == top_key || w >= min_p ? mass_of(w) : 0;
  };
  const uint64_t w_eq = kept_mass(key);
  for (uint32_t i = i0 + lane; i < i1; i += 64) {
    const uint32_t k = key_of((float)x[i]);
    if (k > key)
      mass += kept_mass(k);
    else if (k == key)
      eq++;
  }
  for (int m = 1; m < 64; m <<= 1) {
    mass += __shfl_xor((unsigned long long)mass, m);
    eq += __shfl_xor(eq, m);
  }
  if (lane == 0) {
    slots[wave] = mass;
    slots32[wave] = eq;
  }
  __syncthreads();
  uint64_t total = 0, before = 0;
  uint32_t eq_total = 0, eq_before = 0;
  for (uint32_t i = 0; i < (uint32_t)kWaves; i++) {
    if (i == wave) {
      before = total;
      eq_before = eq_total;
    }
    total += slots[i];
    eq_total += slots32[i];
  }
  auto with_ties = [&](uint64_t m, uint32_t e) { return m + (uint64_t)min(e, ties) * w_eq; };
  const uint64_t all = with_ties(total, eq_total);
  const float u = us[blockIdx.x];
  double goal = u > 0.0f ? (double)u * (double)all : 0.0;
  if (!(goal < (double)all)) goal = (double)(all - 1);
  auto past = [&](uint64_t v) { return (double)v > goal; };
  // the wave whose run crosses the goal finds the index
  if (past(with_ties(before, eq_before)) || !past(with_ties(before + mass, eq_before + eq))) return;
  for (uint32_t b = i0; b < i1; b += 64) {
    const uint32_t i = b + lane;
    const uint32_t k = i < i1 ? key_of((float)x[i]) : 0u;
    uint64_t m = k > key ? kept_mass(k) : 0;
    uint32_t e = k == key ? 1u : 0u;
    for (int w = 1; w < 64; w <<= 1) {
      const uint64_t om = __shfl_up((unsigned long long)m, w);
      const uint32_t oe = __shfl_up(e, w);
      if ((int)lane >= w) {
        m += om;
        e += oe;
      }
    }
    const uint64_t hit = __ballot(past(with_ties(before + m, eq_before + e)));
    if (hit) {
      if (lane == 0) tokens[blockIdx.x] = b + (uint32_t)__builtin_ctzll(hit);
      return;
    }
    before += __shfl((unsigned long long)m, 63);
    eq_before += __shfl(e, 63);
  }
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

uint64_t rlh_sample_rows_workspace(uint64_t n_rows, uint64_t n) {
  (void)n_rows;
  (void)n;
  return 0;
}

int rlh_sample_rows(uint32_t type, const void* logits, uint64_t n_rows, uint64_t n, uint64_t stride,
                    const rlh_row_sampling* options, const float* u, uint32_t* tokens, void* workspace,
                    uint64_t workspace_bytes, void* stream) {
  const uint32_t size = float_type_size(type);
  if (!size) return serve_error(RLH_EUNSUP, "logits are not F32, F16 or BF16");
  if (n == 0 || n > kMaxRow) return serve_error(RLH_EINVAL, "n outside [1, 2^21]");
  if (n_rows > 0x3fffffull) return serve_error(RLH_EUNSUP, "more than 2^22 rows");
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
  const dim3 grid((uint32_t)n_rows);
  if (type == RLH_TYPE_F32)
    hipLaunchKernelGGL(k_sample_row<float>, grid, dim3(kThreads), 0, s, (const float*)logits, n, stride, options, u, tokens);
  else if (type == RLH_TYPE_F16)
    hipLaunchKernelGGL(k_sample_row<_Float16>, grid, dim3(kThreads), 0, s, (const _Float16*)logits, n, stride, options, u, tokens);
  else
    hipLaunchKernelGGL(k_sample_row<__bf16>, grid, dim3(kThreads), 0, s, (const __bf16*)logits, n, stride, options, u, tokens);
  return launched("rlh_sample_rows");
}

}  // extern "C"
