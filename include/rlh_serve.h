/* rlh_serve.h — C ABI of the batched serving operators (MI355X, gfx950).
 *
 * rlh.h runs one sequence per cache, with the reference's bits. The entries
 * here are for a host that serves many sequences at once and owns its
 * memory: a pool of key/value pages, ragged batches of prompts and single
 * tokens, a prefix that the batch shares, and one token drawn per row. They
 * hold f16 or bf16 keys and values and sum in another order than the
 * reference, so they are not bit-compatible with rlh_forward_*.
 *
 * Conventions
 *  - Status codes and rlh_last_error() are those of rlh.h. Arguments are
 *    checked before anything is enqueued: RLH_EINVAL for null, misaligned,
 *    overlapping or contradicting arguments, RLH_EUNSUP for types and sizes
 *    without a kernel. Checks that need no device come first.
 *  - Every pointer is memory that the current device can access, unless it
 *    says host; plain host memory, or memory of another device, is RLH_EINVAL.
 *    Data and workspaces are aligned to 16 bytes, strides count elements and
 *    span a multiple of 16 bytes, index arrays are aligned to 4 bytes, rotary
 *    frequencies to 8. What a call writes overlaps nothing else of it.
 *  - The calls enqueue kernels on `stream` (a hipStream_t of the current device,
 *    NULL for the null stream), allocate nothing and do not synchronize, so they may be captured
 *    into a graph; lengths, positions, page ids and sampling options are read
 *    when the kernels run. Calls that may overlap (two streams, or two
 *    graphs replayed at once) need workspaces of their own; between calls a
 *    workspace holds nothing.
 *  - What the host cannot check, the kernels do, and add a bit to *status
 *    (device memory, may be NULL; never cleared here):
 *    RLH_SERVE_BAD_SEQ: a sequence whose q_start and kv_len contradict each
 *    other or rlh_seqs' bounds is skipped, its rows left as they were;
 *    RLH_SERVE_BAD_PAGE: a page id >= n_pages is neither read nor written, its
 *    positions count as masked.
 */
#ifndef RLH_SERVE_H
#define RLH_SERVE_H

#include "rlh.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RLH_SERVE_BAD_PAGE 1u
#define RLH_SERVE_BAD_SEQ 2u

/* One layer's pool of pages: k and v are [n_pages][n_head_kv][page_size]
 * [head_dim] of `type` (RLH_TYPE_F16 or RLH_TYPE_BF16). head_dim is 64 or
 * 128, page_size a power of two from 16 to 256. */
typedef struct rlh_kv_pages {
  uint32_t type, n_head_kv, head_dim, page_size;
  uint64_t n_pages;
  void* k;
  void* v;
} rlh_kv_pages;

/* A batch: sequence s brings the rows q_start[s] .. q_start[s+1]-1, its last
 * positions: row q_start[s] + i is at position kv_len[s] - new + i, where
 * new = q_start[s+1] - q_start[s] and kv_len[s] counts these rows. Position p
 * lies in page table[s * table_stride + p / page_size], slot p % page_size.
 * q_start (n_seq + 1 values) does not fall; a sequence may bring no rows,
 * and rows before the first or behind the last one are left as they were.
 * max_q and max_kv bound the new rows and kv_len of every sequence (max_kv <=
 * table_stride * page_size < 2^30): work is divided by them, so near bounds are
 * faster.
 * n_seq < 2^16, n_rows <= 2^23, n_rows * n_head <= 2^25 and n_seq * n_head_kv
 * <= 2^21 (RLH_EUNSUP beyond). */
typedef struct rlh_seqs {
  uint32_t n_seq, n_rows, max_q, max_kv, table_stride;
  const uint32_t* q_start;
  const uint32_t* kv_len;
  const uint32_t* table;
} rlh_seqs;

/* ---- rotary positions --------------------------------------------------------
 * Frequencies in radians per position, f_i = theta^(-2i / rot_dim) for
 * i < rot_dim / 2, and the factor of the rotated values (the reference's
 * unscaled table: src/model.rs:700-738 reads theta alone).
 * RLH_ROPE_LINEAR divides every f_i by `factor`. RLH_ROPE_BANDS divides the
 * ones that turn less than beta_slow times over orig_ctx positions, keeps
 * those of more than beta_fast turns, blends linearly in i between, and
 * makes *magnitude 0.1 ln(factor) + 1 (factor >= 1). Host only; `freqs` is
 * host memory of rot_dim / 2 doubles, for the caller to copy to the device. */
#define RLH_ROPE_PLAIN 0u
#define RLH_ROPE_LINEAR 1u
#define RLH_ROPE_BANDS 2u
typedef struct rlh_rope {
  uint32_t rot_dim, scaling;
  double theta, factor, orig_ctx, beta_fast, beta_slow;
} rlh_rope;
int rlh_rope_freqs(const rlh_rope* rope, double* freqs, float* magnitude);

/* ---- append ------------------------------------------------------------------
 * Norms of queries and keys per head, position rotation and the append to
 * the pages in one pass (the reference's rmsnorm_head, RoPE and KV write,
 * src/ops.rs:336-446, for many sequences). q, k and v are rows of in_type
 * (RLH_TYPE_F32, F16 or BF16) with strides of their own, e.g. the slices of
 * one product. q_norm / k_norm (f32[head_dim], each may be NULL):
 * x * w / sqrt(mean(x^2) + eps), the squares summed in f32. The first rot_dim values of a head (a
 * multiple of 16, 0: none) are rotated by position * freqs[i], computed in
 * 64 bits, and multiplied by `magnitude`: pairs (i, i + rot_dim / 2), or
 * (2i, 2i + 1) when `interleaved`. q_out receives the rows of q, k and v
 * pages those of k and v, each rounded once to the pool's type. q_out must
 * not overlap q, k or v. Sequences own the pages that they append to. */
typedef struct rlh_append_args {
  uint32_t in_type, n_head;
  const void* q;
  const void* k;
  const void* v;
  uint64_t q_stride, k_stride, v_stride;
  const float* q_norm;
  const float* k_norm;
  float eps, magnitude;
  const double* freqs;
  uint32_t rot_dim, interleaved;
  void* q_out;
  uint64_t q_out_stride;
} rlh_append_args;
int rlh_paged_append(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_append_args* args, uint32_t* status,
                     void* stream);

/* ---- attention ---------------------------------------------------------------
 * out = softmax(s) V over the positions j that a row at position i sees, for
 * query head h of KV head h / (n_head / n_head_kv):
 *   t = scale * (q . k_j), then softcap * tanh(t / softcap) when softcap > 0
 *   s = t + slopes[h] * (j - i)           when slopes (f32[n_head]) is given
 *   seen: j <= i, and j > i - window when window > 0; and every
 *   j < prefix_len[s] (u32[n_seq], may be NULL), also ahead of i; always
 *   j < kv_len[s]. What is not seen contributes nothing, whatever it holds.
 * The bias is signed as written: a prefix position ahead of a row (j > i) gets
 * slopes[h] times how far ahead it is, not minus that.
 * A row that sees nothing, or only scores of minus infinity, is zero. q and
 * out are [n_rows][n_head][head_dim] of the pool's type with row strides, and
 * must not overlap. Scores, maxima and sums are f32; the probabilities are
 * rounded to the pool's type for the product with V (in f16, those below 2^-21
 * of the largest so far to multiples of 2^-31 of it). A cap of up to 64 puts a
 * score off by 2^-23 of the cap, a larger one by 2^-21 of the score; above 2^100
 * it is taken as 2^100.
 *
 * shared_len > 0 (a multiple of page_size): the first shared_len positions of
 * every sequence lie in the pages of shared_table (u32[shared_len /
 * page_size]) and are read once for the whole batch; the sequences' own
 * table entries before shared_len / page_size are not read.
 *
 * The workspace size follows from the sizes alone (heads, head_dim, n_seq,
 * n_rows, max_q, max_kv, shared_len) and may be 0, as it is for arguments that
 * rlh_paged_attn refuses. It is enough for every call with these heads and n_seq,
 * n_rows, max_q, max_kv and shared_len up to these (a smaller batch may take
 * more than a larger one, as its work is divided into more parts): asked for
 * a host's limits, it is made once. */
typedef struct rlh_attn_args {
  uint32_t n_head, window;
  const void* q;
  void* out;
  uint64_t q_stride, out_stride;
  float scale, softcap;
  const float* slopes;
  const uint32_t* prefix_len;
  const uint32_t* shared_table;
  uint32_t shared_len;
} rlh_attn_args;
uint64_t rlh_paged_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args);
int rlh_paged_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, void* workspace,
                   uint64_t workspace_bytes, uint32_t* status, void* stream);

/* ---- sampling of rows ----------------------------------------------------------
 * One token per row of logits [n_rows][n] (RLH_TYPE_F32, F16 or BF16, aligned
 * to the type only, any row stride), from the caller's random numbers u[row] in [0, 1), with
 * options per row. The filters are rlh_sample's (top-k, then top-p over the
 * softmax of the whole row) and min-p; the draw runs over the kept tokens in
 * index order, so it needs no sorted list:
 *   w_i = exp((l_i - max l) / temperature), in 64 bits, to 2^-37 of itself
 *   order: l descending, equal ones by index
 *   kept: the first top_k (0: all), the shortest head of the order whose
 *   mass reaches top_p * sum(w) (for 0 < top_p < 1), w_i >= min_p (for
 *   min_p > 0); the first of the order is always kept
 *   token: the lowest index whose running kept mass exceeds u * kept mass
 * temperature <= 0 (or NaN): the first of the order. NaN logits have no mass;
 * at +infinity only those logits have; a row without a value above -infinity
 * gives 0. Borders of mass and the draw are met to 2^-36 of sum(w); masses
 * below 2^-43 of the largest may count as none. u outside [0, 1) (or NaN) is
 * taken as the nearer end (0); at 1 and above the token is the last kept one of
 * at least 2^-43 of the largest weight. n <= 2^21, n_rows <= 2^21 and
 * n_rows * n <= 2^35. The token does not depend on the run: masses are summed in
 * a fixed order, or as whole numbers. */
typedef struct rlh_row_sampling {
  float temperature;
  uint32_t top_k;
  float top_p;
  float min_p;
} rlh_row_sampling;
uint64_t rlh_sample_rows_workspace(uint64_t n_rows, uint64_t n);
int rlh_sample_rows(uint32_t type, const void* logits, uint64_t n_rows, uint64_t n, uint64_t stride,
                    const rlh_row_sampling* options, const float* u, uint32_t* tokens, void* workspace,
                    uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RLH_SERVE_H */
