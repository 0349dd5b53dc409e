// Test helper (built by tests/test_cache_edges.py with g++): what
// llama.rs_amd/csrc/paged_index.h says of a drafted row under a window.
#define RLH_HD inline
#include "../llama.rs_amd/csrc/paged_index.h"

extern "C" {

// What a row with this mask sees of positions 0 .. n - 1 where the window bounds the new rows too, as the kernels
// ask for it: by the rows that the window leaves, 64 positions from p on at a time.
void shim_row_sees(const uint64_t* mask, uint32_t words, uint32_t q_len, int32_t first, uint32_t window, uint64_t* left,
                   int32_t p, uint8_t* sees, uint32_t n) {
  if (window != 0 && q_len > window)
    rlh::tree_window(mask, words, q_len, window, left);
  else
    for (uint32_t w = 0; w < words; w++) left[w] = mask[w];
  const rlh::RowSpan r = rlh::tree_span(first, rlh::tree_seen(left, words, q_len), window);
  for (; p < (int32_t)n; p += 64) {
    const uint64_t bits = rlh::tree_bits(left, words, q_len, p - first);
    for (int i = 0; i < 64; i++)
      if (p + i >= 0 && p + i < (int32_t)n) sees[p + i] = rlh::row_sees(r, p + i) || (bits >> i & 1);
  }
}
}
