/* rlh_cache.h — C ABI of the operators that edit a paged cache (MI355X, gfx950).
 *
 * rlh_serve.h appends to a paged key/value cache and attends over it. The
 * entries here are for a host that also takes positions back: one that drafts
 * a tree of tokens per sequence, lets the model judge all of them at once and
 * keeps one branch; and one that drops the positions that got little attention.
 *
 * A step with drafts, for a batch whose rows are the trees' nodes:
 *   rlh_tree_masks       once: who sees whom, and the rotary positions
 *   per layer: rlh_paged_append_at, rlh_tree_attn
 *   rlh_sample_rows      once: a token per node
 *   rlh_tree_accept      once: the branch that the tokens follow
 *   per layer: rlh_paged_move
 * A cache of bounded size, per layer:
 *   rlh_paged_attn_lse   the attention, and the log of each row's sum
 *   rlh_paged_mass       adds each position's attention weights to its mass
 *   rlh_evict_select     when full: the positions that stay
 *   rlh_paged_move       moves them, and their masses, to the front
 *
 * The conventions are those of rlh_serve.h: status codes, checks before
 * anything is enqueued, device memory, alignment, streams, nothing allocated or
 * waited for, what a call writes overlaps nothing else of it unless it says so,
 * and RLH_SERVE_BAD_SEQ / RLH_SERVE_BAD_PAGE in *status. Results do not depend
 * on the run: there are no sums whose order does.
 */
#ifndef RLH_CACHE_H
#define RLH_CACHE_H

#include "rlh_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rows at positions of their own ---------------------------------------------
 * rlh_paged_append with row r rotated by positions[r] (u32[n_rows]) instead of
 * its place in the cache, which stays what seqs says: nodes of a tree, whose
 * place is their number and whose position their depth, and rows behind an
 * eviction. */
int rlh_paged_append_at(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_append_args* args,
                        const uint32_t* positions, uint32_t* status, void* stream);

/* rlh_paged_attn, and lse (f32[n_rows][n_head]): the natural log of the sum of
 * exp(s) over what the row sees, minus infinity where that is nothing. The
 * workspace is rlh_paged_attn's. */
int rlh_paged_attn_lse(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, float* lse,
                       void* workspace, uint64_t workspace_bytes, uint32_t* status, void* stream);

/* ---- trees of drafted tokens ----------------------------------------------------
 * A sequence's new rows are nodes of a tree: parents[row] is the number of
 * the row's parent among the sequence's new rows, smaller than its own, or
 * RLH_NO_PARENT. A number that is not smaller counts as RLH_NO_PARENT, with
 * RLH_SERVE_BAD_SEQ. Only n_seq, n_rows, max_q, max_kv, q_start and kv_len of
 * seqs are read here.
 *
 * masks (u64[n_rows][mask_words], 64 * mask_words >= max_q): bit j % 64 of word
 * j / 64 says that the row sees new row j: itself and its ancestors.
 * positions (u32[n_rows], may be NULL): base[s] (u32[n_seq]; NULL: kv_len - new)
 * plus the row's depth, the number of its ancestors. */
#define RLH_NO_PARENT 0xffffffffu
int rlh_tree_masks(const rlh_seqs* seqs, const uint32_t* parents, const uint32_t* base, uint64_t* masks,
                   uint32_t mask_words, uint32_t* positions, uint32_t* status, void* stream);

/* rlh_paged_attn where a row sees, instead of what comes before it: every
 * position before its sequence's new rows (of which the window, if any, leaves
 * the last window - c, c being the new rows that it sees), and the new rows
 * whose bit its mask has, also behind it; bits of no new row are ignored. Any
 * masks will do, those of rlh_tree_masks among them. The window alone does not
 * bound c: with RLH_WINDOW_DRAFTS | window a row that sees more than `window` new
 * rows sees the last `window` of them (and nothing before), as rlh_paged_attn's
 * row of the same line of tokens does. A model with a window needs it wherever a
 * branch may be longer than the window. (rlh_paged_attn and the entries that
 * score as it does take the flag too: there a window bounds all rows as it is.)
 * slopes and prefix_len are RLH_EUNSUP; shared_len must not reach into the new
 * rows (RLH_SERVE_BAD_SEQ). lse may be NULL. The workspace is as
 * rlh_paged_attn_workspace says of its own; for calls with RLH_WINDOW_DRAFTS it
 * is asked for with it. n_rows * mask_words <= 2^32. */
#define RLH_WINDOW_DRAFTS 0x80000000u
uint64_t rlh_tree_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args);
int rlh_tree_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, const uint64_t* masks,
                  uint32_t mask_words, float* lse, void* workspace, uint64_t workspace_bytes, uint32_t* status,
                  void* stream);

/* The branch of each tree that the model's own tokens follow. A sequence's
 * first new row is the token that the step before ended with: it is always
 * kept. From a kept row r on, the child (the lowest-numbered one) whose drafted
 * token tokens[child] equals sampled[r], the token drawn from row r's logits, is
 * kept next; without one the branch ends there.
 *   path     u32[n_seq][path_stride], path_stride >= max_q: the kept rows'
 *            numbers, ascending; behind count they are left as they were
 *   count    u32[n_seq]: how many; 0 for a sequence without rows or skipped
 *   next     u32[n_seq]: sampled[the last of them]
 *   new_len  u32[n_seq]: kv_len without the rows that are not kept
 * next and new_len are left as they were where count is 0. Parents that are not
 * smaller than their row have no children. seqs is read as above. */
typedef struct rlh_accept_args {
  const uint32_t* parents;
  const uint32_t* tokens;
  const uint32_t* sampled;
  uint32_t* path;
  uint32_t path_stride;
  uint32_t* count;
  uint32_t* next;
  uint32_t* new_len;
} rlh_accept_args;
int rlh_tree_accept(const rlh_seqs* seqs, const rlh_accept_args* args, uint32_t* status, void* stream);

/* ---- moving rows ------------------------------------------------------------------
 * Place base[s] + j of sequence s takes the key and value row of place base[s] +
 * index[j], for all j < count[s] at once: the rows that stay, moved together in
 * place. Lists (u32, index_stride values apart) are per sequence, or with
 * per_head per sequence and KV head. index[j] >= j, in any order, and the same
 * row may be named twice; an entry below its j, or at or past kv_len, moves
 * nothing (RLH_SERVE_BAD_SEQ). count[s] <= max_count <= index_stride, a sequence
 * beyond is skipped; base NULL: 0. mass (f32[n_pages][n_head_kv][page_size], may
 * be NULL) moves along into mass_out, which is mass itself or an array apart
 * (then entries with index[j] = j are copied too). Of seqs n_seq, max_kv,
 * table_stride, kv_len (the lengths before the move) and table are read, n_rows,
 * max_q and q_start are not. Sequences own the pages that change. */
typedef struct rlh_move_args {
  const uint32_t* index;
  uint32_t index_stride, per_head;
  const uint32_t* count;
  uint32_t max_count;
  const uint32_t* base;
  const float* mass;
  float* mass_out;
} rlh_move_args;
int rlh_paged_move(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_move_args* args, uint32_t* status,
                   void* stream);

/* ---- eviction by gathered attention weight ------------------------------------------
 * mass (f32[n_pages][n_head_kv][page_size], beside the pool's rows) holds what
 * each position of each KV head has been attended to. After the attention of
 * `args` and its lse:
 *   mass_j = decay * mass_j + sum over the sequence's new rows i that see j and
 *            the heads h of the KV head's group of exp(s_ijh - lse_ih)
 * for shared_len <= j < kv_len, s as rlh_paged_attn has it (slopes, cap, window
 * and prefix_len as given there; out and shared_table are not read). Of the new
 * rows' own positions, and everywhere with decay 0, the old value is not read.
 * Rows whose lse is minus infinity add nothing. decay is finite and not
 * negative. Scores, exponentials and sums are f32; a term is off by about 2^-21
 * of itself (a score of 16; more for larger ones) and as a cap is in
 * rlh_paged_attn; terms below 2^-126 may count as none. v of kv is not read. Sequences own the pages from shared_len on;
 * a sequence without rows is left alone. */
int rlh_paged_mass(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, const float* lse,
                   float decay, float* mass, uint32_t* status, void* stream);

/* The positions of each sequence and KV head that stay: all if there are at
 * most `budget`; else the first first_kept, the last last_kept and, of those
 * between, the ones of largest mass up to budget in all, equal ones by lowest
 * position (0 and -0 are equal, NaN is below all). keep (u32[n_seq][n_head_kv]
 * [keep_stride]) lists them ascending, behind count as it was; count
 * (u32[n_seq]) is min(kv_len, budget), 0 for a sequence that is skipped:
 * rlh_paged_move's index, per_head, and count. first_kept + last_kept <= budget,
 * keep_stride >= min(budget, max_kv). Positions of pages that do not exist
 * count as NaN. Of seqs n_seq, max_kv, table_stride, kv_len and table are read;
 * of kv the sizes. */
typedef struct rlh_evict_args {
  const float* mass;
  uint32_t budget, first_kept, last_kept, keep_stride;
  uint32_t* keep;
  uint32_t* count;
} rlh_evict_args;
int rlh_evict_select(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_evict_args* args, uint32_t* status,
                     void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RLH_CACHE_H */
