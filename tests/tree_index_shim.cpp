// Test helper (built by tests/test_cache.py with g++): the index rules of
// llama.rs_amd/csrc/paged_index.h for drafted rows, as plain functions.
#define RLH_HD inline
#include "../llama.rs_amd/csrc/paged_index.h"

extern "C" {

// What a row with this mask sees of positions 0 .. n - 1, as the kernels ask for it: 64 positions from p on at a time.
uint32_t shim_tree_sees(const uint64_t* mask, uint32_t words, uint32_t q_len, int32_t first, uint32_t window, int32_t p,
                        uint8_t* sees, uint32_t n) {
  const uint32_t seen = rlh::tree_seen(mask, words, q_len);
  const rlh::RowSpan r = rlh::tree_span(first, seen, window);
  for (; p < (int32_t)n; p += 64) {
    const uint64_t bits = rlh::tree_bits(mask, words, q_len, p - first);
    for (int i = 0; i < 64; i++)
      if (p + i >= 0 && p + i < (int32_t)n) sees[p + i] = rlh::row_sees(r, p + i) || (bits >> i & 1);
  }
  return seen;
}

uint64_t shim_line_units(uint32_t rows, uint32_t steps) { return rlh::line_units(rows, steps); }
uint64_t shim_line_share(uint64_t units, uint32_t blocks) { return rlh::line_share(units, blocks); }
uint32_t shim_line_weight(uint32_t rows) { return rlh::line_weight(rows); }

// The segments of block `block` among tiles that begin at unit `first`: of
// each {tile, first step, end step, slot}. Returns how many.
uint32_t shim_line_block(uint64_t first, uint32_t rows, uint32_t steps, uint64_t share, uint32_t block, uint32_t (*out)[4]) {
  const uint64_t end = first + rlh::line_units(rows, steps), x1 = (block + 1) * share < end ? (block + 1) * share : end;
  uint64_t x = block * share > first ? block * share : first;
  uint32_t n = 0;
  while (x < x1) {
    const uint32_t k = rlh::line_at(first, rows, steps, x);
    const rlh::LineTile t = rlh::line_tile(first, rows, steps, k);
    out[n][0] = k;
    out[n][1] = rlh::line_step(t, x);
    out[n][2] = rlh::line_end(t) <= x1 ? steps : rlh::line_step(t, x1);
    out[n][3] = rlh::line_slot(t, block, share);
    n++;
    x = rlh::line_end(t);
  }
  return n;
}

// Of tile k: the blocks of its first and last step, and the slot of each.
void shim_line_parts(uint64_t first, uint32_t rows, uint32_t steps, uint64_t share, uint32_t k, uint32_t* blocks,
                     uint32_t* slots) {
  const rlh::LineTile t = rlh::line_tile(first, rows, steps, k);
  blocks[0] = rlh::line_first_block(t, share);
  blocks[1] = rlh::line_last_block(t, share);
  for (uint32_t b = blocks[0]; b <= blocks[1]; b++) slots[b - blocks[0]] = rlh::line_slot(t, b, share);
}
}
