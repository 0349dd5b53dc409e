// paged_index.h — what a ragged batch over a paged cache means: which rows
// and positions a sequence has, what a row sees, where a position lies. One
// source for the kernels and for the host test that runs it on bad input.
#pragma once
#include <stdint.h>

#ifndef RLH_HD
#define RLH_HD __host__ __device__ __forceinline__
#endif

namespace rlh {

// One sequence of rlh_seqs. `ok` is false for one that is skipped.
struct SeqView {
  uint32_t q0;      // first row
  uint32_t q_len;   // new rows
  uint32_t kv_len;  // positions, the new rows included
  bool ok;
};

// a = q_start[s], b = q_start[s + 1]. A sequence without rows is not an error
// whatever its length says (padding of a batch).
RLH_HD SeqView seq_view(uint32_t a, uint32_t b, uint32_t kv, uint32_t n_rows, uint32_t max_q, uint32_t max_kv,
                        bool* bad) {
  SeqView v;
  v.q0 = a;
  v.q_len = b - a;
  v.kv_len = kv;
  v.ok = a < b && b <= n_rows && b - a <= max_q && kv <= max_kv && b - a <= kv;
  *bad = !v.ok && a != b;
  return v;
}

// The positions a row sees are [lo, hi) below its sequence's length, where
// with a prefix those of [0, prefix) are added (prefix <= hi after
// clamping); window 0 means none.
struct RowSpan {
  int32_t lo, hi, prefix;
};

RLH_HD RowSpan row_span(int32_t pos, uint32_t kv_len, uint32_t window, uint32_t prefix) {
  RowSpan r;
  r.hi = pos + 1;
  r.lo = window != 0 && (uint32_t)pos >= window ? pos - (int32_t)window + 1 : 0;
  r.prefix = (int32_t)(prefix < kv_len ? prefix : kv_len);
  return r;
}

// (no short-circuits: the kernels ask for every score of a border tile)
RLH_HD bool row_sees(const RowSpan& r, int32_t j) { return ((j >= r.lo) & (j < r.hi)) | (j < r.prefix); }

// First and end position that any row of positions [first, last] sees (with
// both a prefix and a window, what lies between them is stepped through).
RLH_HD int32_t span_begin(const RowSpan& first) { return first.prefix > 0 ? 0 : first.lo; }
RLH_HD int32_t span_end(const RowSpan& last) { return last.hi > last.prefix ? last.hi : last.prefix; }

// Steps of an item when the `steps` of all sequences (fewer than 2^24 each, so
// that 32 bits hold the sum of 256 of them, not of 65535) are divided into
// `goal` items: the sequences' own, rounded up, are at most `goal` and one each.
RLH_HD uint32_t steps_per_item(uint64_t steps, uint32_t goal) {
  const uint64_t n = (steps + goal - 1) / goal;
  return n < 1u << 24 ? (uint32_t)n : 1u << 24;
}
RLH_HD uint32_t items_of(uint32_t steps, uint32_t per_item) { return (steps + per_item - 1) / per_item; }

}  // namespace rlh
