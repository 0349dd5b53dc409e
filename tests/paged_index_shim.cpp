// Test helper (built by tests/test_serve.py with g++): the index rules of
// llama.rs_amd/csrc/paged_index.h as plain functions.
#define RLH_HD inline
#include "../llama.rs_amd/csrc/paged_index.h"

extern "C" {

int shim_seq_view(uint32_t a, uint32_t b, uint32_t kv, uint32_t n_rows, uint32_t max_q, uint32_t max_kv, uint32_t* out) {
  bool bad;
  const rlh::SeqView v = rlh::seq_view(a, b, kv, n_rows, max_q, max_kv, &bad);
  out[0] = v.q0;
  out[1] = v.q_len;
  out[2] = v.kv_len;
  return (v.ok ? 1 : 0) | (bad ? 2 : 0);
}

// sees[j] for j < n, and the tile range of rows first..last
void shim_sees(int32_t pos, uint32_t kv_len, uint32_t window, uint32_t prefix, uint8_t* sees, uint32_t n) {
  const rlh::RowSpan r = rlh::row_span(pos, kv_len, window, prefix);
  for (uint32_t j = 0; j < n; j++) sees[j] = rlh::row_sees(r, (int32_t)j);
}

void shim_range(int32_t first, int32_t last, uint32_t kv_len, uint32_t window, uint32_t prefix, int32_t* out) {
  out[0] = rlh::span_begin(rlh::row_span(first, kv_len, window, prefix));
  out[1] = rlh::span_end(rlh::row_span(last, kv_len, window, prefix));
}
}
