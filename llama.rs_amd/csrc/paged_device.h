// paged_device.h — device helpers shared by the kernels over the paged cache.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_index.h"

namespace rlh {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// One batch as the kernels get it.
struct Batch {
  uint32_t n_seq, n_rows, max_q, max_kv, table_stride;
  const uint32_t* q_start;
  const uint32_t* kv_len;
  const uint32_t* table;
};

__device__ __forceinline__ SeqView load_seq(const Batch& b, uint32_t s, bool* bad) {
  return seq_view(b.q_start[s], b.q_start[s + 1], b.kv_len[s], b.n_rows, b.max_q, b.max_kv, bad);
}

__device__ __forceinline__ void raise(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

// How many of the n values a[0], a[stride], ... that do not fall are at most x:
// a wave's 64 lanes try places of the range that is left. (Ends within [0, n]
// also where they fall.)
__device__ __forceinline__ uint32_t count_upto(const uint32_t* a, uint32_t stride, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t step = (hi - lo + 63) / 64, i = lo + (threadIdx.x & 63) * step;
    const uint64_t above = ~__ballot(i < hi && a[(size_t)i * stride] <= x);
    const uint32_t f = above ? (uint32_t)__builtin_ctzll(above) : 64u;  // places from the first on that are not above
    if (f == 0) break;
    hi = min(hi, lo + f * step);
    lo += (f - 1) * step + 1;
  }
  return lo;
}

}  // namespace rlh
