// paged_attn.hip — attention of a ragged batch over the paged cache.
#include <math.h>

#include "paged_device.h"
#include "serve_check.h"

namespace rlh {
namespace {

struct AttnParams {
  Batch b;
  const void *q, *pool_k, *pool_v;
  void* out;
  uint64_t q_stride, out_stride;
  const float* slopes;
  const uint32_t *prefix_len, *shared_table;
  uint32_t* status;
  float scale, softcap;
  uint32_t n_head, n_kv, group, page_shift, n_pages, window, shared_len;
};

constexpr float kLog2e = 1.4426950408889634f;

// Whole workgroup: the sequence that row `row` belongs to (n_seq: none).
__device__ __forceinline__ uint32_t block_seq_of(const Batch& b, uint32_t row) {
  uint32_t s = 0;
  for (uint32_t i = 0; i < b.n_seq; i += blockDim.x) {
    const uint32_t k = i + threadIdx.x;
    s += (uint32_t)__syncthreads_count(k < b.n_seq && b.q_start[k + 1] <= row);
  }
  return s;
}

// One wave per (row, query head): 64 positions at a time.
template <typename T, int D>
__global__ void __launch_bounds__(64) k_attn_rows(AttnParams a) {
  __shared__ float qs[D];
  const uint32_t row = blockIdx.x, h = blockIdx.y, g = h / a.group;
  const uint32_t s = block_seq_of(a.b, row);
  if (s >= a.b.n_seq) return;
  bool bad;
  const SeqView sv = load_seq(a.b, s, &bad);
  if (!sv.ok || row < sv.q0) {
    if (threadIdx.x == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
    return;
  }
  const int lane = threadIdx.x;
  const int32_t pos = (int32_t)(sv.kv_len - sv.q_len + (row - sv.q0));
  const RowSpan span = row_span(pos, sv.kv_len, a.window, a.prefix_len ? a.prefix_len[s] : 0);
  for (int d = lane; d < D; d += 64) qs[d] = (float)((const T*)a.q)[(size_t)row * a.q_stride + (size_t)h * D + d];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[D / 64] = {};
  for (int32_t j0 = span_begin(span); j0 < span_end(span); j0 += 64) {
    const int32_t j = j0 + lane;
    bool see = j < (int32_t)sv.kv_len && row_sees(span, j);
    uint32_t page = 0;
    if (see) {
      page = j < (int32_t)a.shared_len ? a.shared_table[j >> a.page_shift]
                                       : a.b.table[(size_t)s * a.b.table_stride + (j >> a.page_shift)];
      if (page >= a.n_pages) {
        raise(a.status, RLH_SERVE_BAD_PAGE);
        see = false;
      }
    }
    const uint32_t slot = j & ((1u << a.page_shift) - 1);
    const size_t at = see ? ((((size_t)page * a.n_kv + g) << a.page_shift) + slot) * D : 0;
    float x = -INFINITY;
    if (see) {
      x = 0.0f;
      for (int d = 0; d < D; d++) x = fmaf(qs[d], (float)((const T*)a.pool_k)[at + d], x);
      x *= a.scale;
      if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
      if (a.slopes) x = fmaf(a.slopes[h], (float)(j - pos), x);
    }
    float mx = x;
    for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
    const float p = exp2f((x - base) * kLog2e), f = exp2f((m - base) * kLog2e);
    float sum = p;
    for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);
    l = l * f + sum;
    m = mn;
    for (int i = 0; i < D / 64; i++) o[i] *= f;
    for (int k = 0; k < 64; k++) {
      const float pk = __shfl(p, k);
      if (!__shfl((int)see, k)) continue;
      const size_t ak = (size_t)__shfl((unsigned long long)at, k);
      for (int i = 0; i < D / 64; i++) o[i] = fmaf(pk, (float)((const T*)a.pool_v)[ak + i * 64 + lane], o[i]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int i = 0; i < D / 64; i++)
    ((T*)a.out)[(size_t)row * a.out_stride + (size_t)h * D + i * 64 + lane] = (T)(o[i] * inv);
}

int check_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  if (!args) return serve_error(RLH_EINVAL, "null argument");
  RLH_TRY(check_batch(kv, seqs, args->n_head));
  if (!isfinite(args->scale)) return serve_error(RLH_EINVAL, "scale is not finite");
  if (!(args->softcap >= 0.0f) || !isfinite(args->softcap)) return serve_error(RLH_EINVAL, "softcap is negative or not finite");
  if (args->shared_len % kv->page_size) return serve_error(RLH_EINVAL, "shared_len is not a multiple of page_size");
  if (args->shared_len >= (1u << 30)) return serve_error(RLH_EUNSUP, "shared_len of 2^30 or more");
  if (args->shared_len && !args->shared_table) return serve_error(RLH_EINVAL, "shared_table is null");
  if (!aligned(args->slopes, 4) || !aligned(args->prefix_len, 4) || !aligned(args->shared_table, 4))
    return serve_error(RLH_EINVAL, "slopes, prefix_len or shared_table is not aligned to 4 bytes");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  const uint64_t w = (uint64_t)args->n_head * kv->head_dim;
  RLH_TRY(check_rows("q", args->q, args->q_stride, w, 2));
  RLH_TRY(check_rows("out", args->out, args->out_stride, w, 2));
  if (overlap(args->q, row_bytes_span(seqs->n_rows, args->q_stride, w, 2), args->out,
              row_bytes_span(seqs->n_rows, args->out_stride, w, 2)))
    return serve_error(RLH_EINVAL, "out overlaps q");
  return RLH_OK;
}

uint64_t attn_workspace(const rlh_kv_pages&, const rlh_seqs&, const rlh_attn_args&) { return 0; }

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

uint64_t rlh_paged_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  if (check_attn(kv, seqs, args) != RLH_OK || seqs->n_seq == 0 || seqs->n_rows == 0) return 0;
  return attn_workspace(*kv, *seqs, *args);
}

int rlh_paged_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, void* workspace,
                   uint64_t workspace_bytes, uint32_t* status, void* stream) {
  RLH_TRY(check_attn(kv, seqs, args));
  if (!aligned(status, 4)) return serve_error(RLH_EINVAL, "status is not aligned to 4 bytes");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  const uint64_t need = attn_workspace(*kv, *seqs, *args);
  if (need && !workspace) return serve_error(RLH_EINVAL, "workspace is null");
  if (need > workspace_bytes)
    return serve_error(RLH_EINVAL, "workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(need) + " needed");
  if (need && !aligned(workspace, 16)) return serve_error(RLH_EINVAL, "workspace is not aligned to 16 bytes");
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("k pages", kv->k));
  RLH_TRY(dev("v pages", kv->v));
  RLH_TRY(dev("q_start", seqs->q_start));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("table", seqs->table));
  RLH_TRY(dev("q", args->q));
  RLH_TRY(dev("out", args->out));
  RLH_TRY(dev("slopes", args->slopes));
  RLH_TRY(dev("prefix_len", args->prefix_len));
  if (args->shared_len) RLH_TRY(dev("shared_table", args->shared_table));
  if (need) RLH_TRY(dev("workspace", workspace));
  RLH_TRY(dev("status", status));
  AttnParams p{};
  p.b = Batch{seqs->n_seq, seqs->n_rows, seqs->max_q, seqs->max_kv, seqs->table_stride,
              seqs->q_start, seqs->kv_len, seqs->table};
  p.q = args->q;
  p.out = args->out;
  p.pool_k = kv->k;
  p.pool_v = kv->v;
  p.q_stride = args->q_stride;
  p.out_stride = args->out_stride;
  p.slopes = args->slopes;
  p.prefix_len = args->prefix_len;
  p.shared_table = args->shared_table;
  p.status = status;
  p.scale = args->scale;
  p.softcap = args->softcap;
  p.n_head = args->n_head;
  p.n_kv = kv->n_head_kv;
  p.group = args->n_head / kv->n_head_kv;
  p.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  p.n_pages = (uint32_t)kv->n_pages;
  p.window = args->window;
  p.shared_len = args->shared_len;
  const dim3 grid(seqs->n_rows, args->n_head);
  hipStream_t s = (hipStream_t)stream;
  const bool f16 = kv->type == RLH_TYPE_F16;
  if (kv->head_dim == 64) {
    if (f16)
      hipLaunchKernelGGL((k_attn_rows<_Float16, 64>), grid, dim3(64), 0, s, p);
    else
      hipLaunchKernelGGL((k_attn_rows<__bf16, 64>), grid, dim3(64), 0, s, p);
  } else {
    if (f16)
      hipLaunchKernelGGL((k_attn_rows<_Float16, 128>), grid, dim3(64), 0, s, p);
    else
      hipLaunchKernelGGL((k_attn_rows<__bf16, 128>), grid, dim3(64), 0, s, p);
  }
  return launched("rlh_paged_attn");
}

}  // extern "C"
