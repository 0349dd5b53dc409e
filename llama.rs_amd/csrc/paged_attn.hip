// paged_attn.hip — attention of a ragged batch over the paged cache: each row
// sees what comes before it.
#include "../../include/rlh_cache.h"
#include "paged_attn.h"

using namespace rlh;

extern "C" {

uint64_t rlh_paged_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  if (check_attn(kv, seqs, args) != RLH_OK || seqs->n_seq == 0 || seqs->n_rows == 0) return 0;
  return attn_workspace<false>(*kv, *seqs, *args);
}

int rlh_paged_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, void* workspace,
                   uint64_t workspace_bytes, uint32_t* status, void* stream) {
  RLH_TRY(check_attn(kv, seqs, args));
  return run_attn<false>("rlh_paged_attn", kv, seqs, args, nullptr, 0, nullptr, workspace, workspace_bytes, status, stream);
}

int rlh_paged_attn_lse(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, float* lse,
                       void* workspace, uint64_t workspace_bytes, uint32_t* status, void* stream) {
  RLH_TRY(check_attn(kv, seqs, args));
  if (!lse && seqs->n_seq != 0 && seqs->n_rows != 0) return serve_error(RLH_EINVAL, "lse is null");
  return run_attn<false>("rlh_paged_attn_lse", kv, seqs, args, nullptr, 0, lse, workspace, workspace_bytes, status, stream);
}

}  // extern "C"
