// Test helper (built by tests/test_serve_edges.py with g++): how
// llama.rs_amd/csrc/paged_index.h divides the work of many sequences.
#define RLH_HD inline
#include "../llama.rs_amd/csrc/paged_index.h"

extern "C" {

// Items that sequences of steps[i] steps, times[i] of each, are divided into.
uint64_t shim_items(const uint32_t* steps, const uint32_t* times, uint32_t n, uint32_t goal, uint32_t* per_item) {
  uint64_t all = 0, items = 0;
  for (uint32_t i = 0; i < n; i++) all += (uint64_t)steps[i] * times[i];
  *per_item = rlh::steps_per_item(all, goal);
  for (uint32_t i = 0; i < n; i++) items += (uint64_t)rlh::items_of(steps[i], *per_item) * times[i];
  return items;
}
}
