// tree_attn.hip — attention of drafted rows over the paged cache: each sees the
// positions before its batch and, by bitmask, rows of the batch itself. The
// kernels are those of paged_attn.h; only steps at a window's start and over the
// new rows ask which score counts, all others run as a prompt's do.
#include "../../include/rlh_cache.h"
#include "paged_attn.h"

using namespace rlh;

namespace {

int check_tree(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  RLH_TRY(check_attn(kv, seqs, args));
  if (args->slopes) return serve_error(RLH_EUNSUP, "slopes: a tree has no distances");
  if (args->prefix_len) return serve_error(RLH_EUNSUP, "prefix_len: what drafted rows see of each other is in the masks");
  return RLH_OK;
}

}  // namespace

extern "C" {

uint64_t rlh_tree_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  if (check_tree(kv, seqs, args) != RLH_OK || seqs->n_seq == 0 || seqs->n_rows == 0) return 0;
  return attn_workspace<true>(*kv, *seqs, *args);
}

int rlh_tree_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, const uint64_t* masks,
                  uint32_t mask_words, float* lse, void* workspace, uint64_t workspace_bytes, uint32_t* status,
                  void* stream) {
  RLH_TRY(check_tree(kv, seqs, args));
  if (seqs->n_seq != 0 && seqs->n_rows != 0) {
    if (!masks || !aligned(masks, 8)) return serve_error(RLH_EINVAL, "masks is null or not aligned to 8 bytes");
    if ((uint64_t)mask_words * 64 < seqs->max_q) return serve_error(RLH_EINVAL, "mask_words holds fewer than max_q bits");
    if ((uint64_t)seqs->n_rows * mask_words > (1ull << 32)) return serve_error(RLH_EUNSUP, "n_rows * mask_words above 2^32");
  }
  return run_attn<true>("rlh_tree_attn", kv, seqs, args, masks, mask_words, lse, workspace, workspace_bytes, status, stream);
}

}  // extern "C"
