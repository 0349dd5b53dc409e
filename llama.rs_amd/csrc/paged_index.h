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

// ---- drafted rows -----------------------------------------------------------------
// What a drafted row sees before its batch, whose first position is `first`: with
// a window, `seen` (the new rows that it sees) take their part of it. lo may be
// past hi: then nothing.
RLH_HD RowSpan tree_span(int32_t first, uint32_t seen, uint32_t window) {
  RowSpan r;
  const uint64_t end = (uint64_t)(uint32_t)first + seen;
  r.hi = first;
  r.lo = window != 0 && end > window ? (int32_t)(end - window) : 0;
  r.prefix = 0;
  return r;
}

// The low `rows` bits of x.
RLH_HD uint64_t only_rows(uint64_t x, int64_t rows) { return rows <= 0 ? 0 : rows >= 64 ? x : x & ((1ull << rows) - 1); }

// New rows that a mask of `words` words names.
RLH_HD uint32_t tree_seen(const uint64_t* mask, uint32_t words, uint32_t q_len) {
  uint32_t n = 0;
  for (uint32_t w = 0; w < words && w * 64 < q_len; w++)
    n += (uint32_t)__builtin_popcountll(only_rows(mask[w], (int64_t)q_len - w * 64));
  return n;
}

// Bits off .. off + 63 of the mask (off may lie before or behind it).
RLH_HD uint64_t tree_bits(const uint64_t* mask, uint32_t words, uint32_t q_len, int32_t off) {
  if (off <= -64 || off >= (int32_t)q_len) return 0;
  const int32_t w = off >> 6;  // floor
  const uint32_t sh = (uint32_t)off & 63;
  const uint64_t a = w >= 0 && (uint32_t)w < words ? mask[w] : 0;
  const uint64_t b = w + 1 >= 0 && (uint32_t)(w + 1) < words && sh ? mask[w + 1] : 0;
  const uint64_t x = sh ? a >> sh | b << (64 - sh) : a;
  return only_rows(x, (int64_t)q_len - off);
}

// The last `window` of the new rows that a mask names, as a mask of as many words.
RLH_HD void tree_window(const uint64_t* mask, uint32_t words, uint32_t q_len, uint32_t window, uint64_t* out) {
  uint32_t left = window;
  for (uint32_t w = words; w-- > 0;) {
    uint64_t x = only_rows(mask[w], (int64_t)q_len - (int64_t)w * 64);
    uint32_t n = (uint32_t)__builtin_popcountll(x);
    for (; n > left; n--) x &= x - 1;
    left -= n;
    out[w] = x;
  }
}

// ---- a line of tiles ------------------------------------------------------------------
// The work of drafted rows: tiles of up to kLineRows rows of a KV head, each of
// which takes the same `steps`; all tiles, one behind the other, make a line that
// blocks share equally, so that a block may end inside a tile and go on
// with the next. Lengths are in units: a step of a tile of more than half the
// rows takes three, of another two (there one of a SIMD's two waves idles and
// memory sets the pace: 2.1 to 2.3 us, and 1.5 to 1.7), a tile's start two steps more.
constexpr uint32_t kLineRows = 256;
constexpr uint32_t kLineStart = 2;
// Units of a block at least: a step, so that the blocks of a tile follow one on
// another. (A block starts with a chain of loads that takes as long as five
// steps, but the starts of blocks that would otherwise not be there cost nothing:
// a tree of 26 nodes at 640 positions takes 14 us, by blocks of at least 12 units 19.)
constexpr uint32_t kLineLeast = 4;

// a / b, by 32 bits where they do (64 take some 200 instructions more).
RLH_HD uint64_t line_div(uint64_t a, uint64_t b) {
  return ((a | b) >> 32) == 0 ? (uint64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
RLH_HD uint32_t line_weight(uint32_t rows) { return rows > kLineRows / 2 ? 3 : 2; }
RLH_HD uint32_t line_tiles(uint32_t rows) { return (rows + kLineRows - 1) / kLineRows; }
// Units of all tiles of `rows` rows.
RLH_HD uint64_t line_units(uint32_t rows, uint32_t steps) {
  if (rows == 0) return 0;
  const uint32_t full = line_tiles(rows) - 1;
  return ((uint64_t)full * 3 + line_weight(rows - full * kLineRows)) * (steps + kLineStart);
}
RLH_HD uint64_t line_share(uint64_t units, uint32_t blocks) {
  const uint64_t n = line_div(units + blocks - 1, blocks);
  return n > kLineLeast ? n : kLineLeast;
}

// Tile k of `rows` rows whose first tile begins at unit `first`.
struct LineTile {
  uint64_t begin;  // unit
  uint32_t weight, steps;
};
RLH_HD LineTile line_tile(uint64_t first, uint32_t rows, uint32_t steps, uint32_t k) {
  return LineTile{first + (uint64_t)k * 3 * (steps + kLineStart), line_weight(rows - k * kLineRows), steps};
}
RLH_HD uint64_t line_end(const LineTile& t) { return t.begin + (uint64_t)t.weight * (t.steps + kLineStart); }
// The tile that unit x, at or behind `first`, lies in.
RLH_HD uint32_t line_at(uint64_t first, uint32_t rows, uint32_t steps, uint64_t x) {
  if (rows <= kLineRows) return 0;
  const uint64_t k = line_div(x - first, 3 * (uint64_t)(steps + kLineStart));
  return k < line_tiles(rows) ? (uint32_t)k : line_tiles(rows) - 1;
}
// A step belongs to the block in whose units it begins: the first step that
// begins at unit x or behind, and the blocks (of `share` units, more than a
// step's) of the first and the last one.
RLH_HD uint32_t line_step(const LineTile& t, uint64_t x) {
  // (fewer than 2^26 units, or the tile is over)
  const uint64_t u = x > t.begin ? x - t.begin : 0;
  if (u >= (uint64_t)t.weight * (t.steps + kLineStart)) return t.steps;
  const uint32_t n = t.weight == 2 ? ((uint32_t)u + 1) / 2 : ((uint32_t)u + 2) / 3;
  return n <= kLineStart ? 0 : n - kLineStart < t.steps ? n - kLineStart : t.steps;
}
RLH_HD uint32_t line_first_block(const LineTile& t, uint64_t share) {
  return (uint32_t)line_div(t.begin + t.weight * kLineStart, share);
}
RLH_HD uint32_t line_last_block(const LineTile& t, uint64_t share) {
  return (uint32_t)line_div(t.begin + (uint64_t)t.weight * (kLineStart + t.steps - 1), share);
}
// A block has two places for parts of tiles: the first for the tile that it
// begins in or at, the second for one that it begins and does not end.
RLH_HD uint32_t line_slot(const LineTile& t, uint32_t block, uint64_t share) {
  return 2 * block + (block * share < t.begin ? 1 : 0);
}

// Steps of an item when the `steps` of all sequences (fewer than 2^24 each, so
// that 32 bits hold the sum of 256 of them, not of 65535) are divided into
// `goal` items: the sequences' own, rounded up, are at most `goal` and one each.
RLH_HD uint32_t steps_per_item(uint64_t steps, uint32_t goal) {
  const uint64_t n = (steps + goal - 1) / goal;
  return n < 1u << 24 ? (uint32_t)n : 1u << 24;
}
RLH_HD uint32_t items_of(uint32_t steps, uint32_t per_item) { return (steps + per_item - 1) / per_item; }

}  // namespace rlh
