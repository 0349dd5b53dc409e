// paged.hip — the paged key/value cache: argument checks that its operators
// share, rotary frequencies, and the append (norms of queries and keys per
// head, position rotation, write to the pages) in one pass.
#include <math.h>

#include "../../include/rlh_cache.h"
#include "paged_device.h"
#include "serve_check.h"

namespace rlh {

int check_batch(const rlh_kv_pages* kv, const rlh_seqs* seqs, uint32_t n_head) {
  if (!kv || !seqs) return serve_error(RLH_EINVAL, "null argument");
  if (kv->type != RLH_TYPE_F16 && kv->type != RLH_TYPE_BF16)
    return serve_error(RLH_EUNSUP, "pages hold F16 or BF16, not type " + std::to_string(kv->type));
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return serve_error(RLH_EUNSUP, "head_dim " + std::to_string(kv->head_dim) + " (64 or 128)");
  if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
    return serve_error(RLH_EUNSUP, "page_size " + std::to_string(kv->page_size) + " (a power of two from 16 to 256)");
  if (n_head == 0 || kv->n_head_kv == 0 || n_head % kv->n_head_kv)
    return serve_error(RLH_EINVAL, "n_head is not a multiple of n_head_kv");
  if (n_head > 1024) return serve_error(RLH_EUNSUP, "more than 1024 query heads");
  if (kv->n_pages == 0 || kv->n_pages > 0x7fffffffull) return serve_error(RLH_EINVAL, "n_pages out of range");
  if (!kv->k || !kv->v) return serve_error(RLH_EINVAL, "the pool's k or v is null");
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return serve_error(RLH_EINVAL, "the pool is not aligned to 16 bytes");
  const uint64_t pool = pool_bytes(*kv);
  if (overlap(kv->k, pool, kv->v, pool)) return serve_error(RLH_EINVAL, "the pool's k and v overlap");
  if (seqs->n_seq > 65535) return serve_error(RLH_EUNSUP, "more than 65535 sequences");
  if (seqs->n_rows > 0x800000u) return serve_error(RLH_EUNSUP, "more than 2^23 rows");
  // launches hold fewer than 2^24 blocks of 256 threads
  if ((uint64_t)seqs->n_rows * n_head > (1ull << 25)) return serve_error(RLH_EUNSUP, "n_rows * n_head above 2^25");
  if ((uint64_t)seqs->n_seq * kv->n_head_kv > (1ull << 21)) return serve_error(RLH_EUNSUP, "n_seq * n_head_kv above 2^21");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;  // nothing to do
  if (!seqs->q_start || !seqs->kv_len || !seqs->table) return serve_error(RLH_EINVAL, "a batch array is null");
  if (!aligned(seqs->q_start, 4) || !aligned(seqs->kv_len, 4) || !aligned(seqs->table, 4))
    return serve_error(RLH_EINVAL, "a batch array is not aligned to 4 bytes");
  if (seqs->max_q == 0 || seqs->max_q > seqs->n_rows) return serve_error(RLH_EINVAL, "max_q outside [1, n_rows]");
  const uint64_t reach = (uint64_t)seqs->table_stride * kv->page_size;
  if (reach >= (1ull << 30)) return serve_error(RLH_EUNSUP, "the table reaches 2^30 positions");
  if (seqs->max_kv < seqs->max_q || seqs->max_kv > reach)
    return serve_error(RLH_EINVAL, "max_kv outside [max_q, table_stride * page_size]");
  return RLH_OK;
}

namespace {

// ---- append ---------------------------------------------------------------------
// Eight values of a head per lane: 16 (head_dim 128) or 8 lanes hold a head,
// a block of 256 threads 16 or 32 heads of one row; a norm's sum and a
// rotation's partners are exchanged between a head's lanes, so that every value
// is read and written once. Bound by HBM for prompts (9503 f32 rows of 64 + 16
// heads: 584 MB in 119 us, 4.9 TB/s; a copy of 2 GiB moves 5.1) and by launch
// latency for single tokens (93 rows: 3.9 us). Norms and rotations are f32,
// angles are reduced in 64 bits; each result is rounded once.

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4_t a = *(const f32x4_t*)p, b = *(const f32x4_t*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    typedef T V8 __attribute__((ext_vector_type(8)));
    const V8 a = *(const V8*)p;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)a[i];
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  typedef T V8 __attribute__((ext_vector_type(8)));
  V8 a;
#pragma unroll
  for (int i = 0; i < 8; i++) a[i] = (T)x[i];
  *(V8*)p = a;
}

struct AppendParams {
  Batch b;
  const void *q, *k, *v;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;
  const float *q_norm, *k_norm;
  const double* freqs;
  const uint32_t* positions;  // rotary, per row; null: the rows' places
  float eps, magnitude;
  uint32_t n_head, n_kv, page_shift, n_pages, rot_dim;
  void *q_out, *pool_k, *pool_v;
  uint32_t* status;
};

template <typename TI, typename TO, int D, bool INTER>
__global__ void __launch_bounds__(kThreads) k_paged_append(AppendParams a) {
  constexpr int L = D / 8;           // lanes per head
  constexpr int HB = kThreads / L;   // heads per block
  __shared__ float cs[D / 2], sn[D / 2];
  const uint32_t row = blockIdx.x;
  // the row's sequence: as many end at or before it as come before it
  uint32_t s = 0;
  if (a.b.n_seq <= kThreads) {
    const uint32_t k = threadIdx.x;
    s = (uint32_t)__syncthreads_count(k < a.b.n_seq && a.b.q_start[k + 1] <= row);
  } else {
    s = count_upto(a.b.q_start + 1, 1, a.b.n_seq, row);
  }
  if (s >= a.b.n_seq) return;  // behind the last sequence
  bool bad;
  const SeqView sv = load_seq(a.b, s, &bad);
  if (s == 0 && !bad && row < sv.q0) return;  // before the first sequence
  if (!sv.ok || row < sv.q0 || row - sv.q0 >= sv.q_len) {  // (starts that fall may name a sequence that ends before it)
    if (threadIdx.x == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
    return;
  }
  const uint32_t pos = sv.kv_len - sv.q_len + (row - sv.q0);
  const uint32_t half = a.rot_dim / 2;
  if (threadIdx.x < half) {
    // turns in 64 bits: at a position of 10^6 an f32 angle is off by 0.03
    const double turns = (double)(a.positions ? a.positions[row] : pos) * a.freqs[threadIdx.x] * 0.15915494309189535;
    const float f = (float)(turns - rint(turns));
    float sv_, cv_;
    sincospif(2.0f * f, &sv_, &cv_);
    cs[threadIdx.x] = cv_ * a.magnitude;
    sn[threadIdx.x] = sv_ * a.magnitude;
  }
  __syncthreads();
  const uint32_t c = threadIdx.x % L;                               // chunk of the head
  const uint32_t head = blockIdx.y * HB + threadIdx.x / L;          // q heads, then k, then v
  const uint32_t H = a.n_head, G = a.n_kv;
  if (head >= H + 2 * G) return;  // whole heads leave: the exchanges below stay within a head
  const bool is_q = head < H, is_k = !is_q && head < H + G;
  const uint32_t hl = is_q ? head : is_k ? head - H : head - H - G;
  const TI* src = is_q ? (const TI*)a.q + (size_t)row * a.q_stride
                       : is_k ? (const TI*)a.k + (size_t)row * a.k_stride : (const TI*)a.v + (size_t)row * a.v_stride;
  float x[8];
  load8(src + (size_t)hl * D + c * 8, x);
  if (is_q || is_k) {
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (w) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int m = 1; m < L; m <<= 1) ss += __shfl_xor(ss, m);
      const float r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      float wv[8];
      load8(w + c * 8, wv);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = x[i] * r * wv[i];
    }
    if constexpr (INTER) {
      if (c < a.rot_dim / 8) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float co = cs[c * 4 + i], si = sn[c * 4 + i], u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = u * co - v * si;
          x[2 * i + 1] = v * co + u * si;
        }
      }
    } else {
      const uint32_t hc = a.rot_dim / 16;  // chunks of a half
      const bool low = c < hc, rot = c < 2 * hc;
      const int from = (int)((threadIdx.x & 63) - c + (low ? c + hc : rot ? c - hc : c));
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = __shfl(x[i], from);
      if (rot) {
        const uint32_t p = (low ? c : c - hc) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float si = low ? -sn[p + i] : sn[p + i];
          x[i] = x[i] * cs[p + i] + y[i] * si;
        }
      }
    }
  }
  if (is_q) {
    store8((TO*)a.q_out + (size_t)row * a.q_out_stride + (size_t)hl * D + c * 8, x);
    return;
  }
  const uint32_t page = a.b.table[(size_t)s * a.b.table_stride + (pos >> a.page_shift)];
  if (page >= a.n_pages) {
    raise(a.status, RLH_SERVE_BAD_PAGE);
    return;
  }
  const uint32_t slot = pos & ((1u << a.page_shift) - 1);
  TO* pool = (TO*)(is_k ? a.pool_k : a.pool_v);
  store8(pool + ((((size_t)page * G + hl) << a.page_shift) + slot) * D + c * 8, x);
}

template <typename TI, typename TO, int D>
int launch_append(const AppendParams& p, bool inter, hipStream_t s) {
  const uint32_t per = kThreads / (D / 8);
  const dim3 grid(p.b.n_rows, (p.n_head + 2 * p.n_kv + per - 1) / per);
  const auto kernel = inter ? k_paged_append<TI, TO, D, true> : k_paged_append<TI, TO, D, false>;
  return enqueue("rlh_paged_append", kernel, grid, kThreads, 0, s, p);
}

template <typename TI, typename TO>
int launch_append(const AppendParams& p, uint32_t dim, bool inter, hipStream_t s) {
  return dim == 64 ? launch_append<TI, TO, 64>(p, inter, s) : launch_append<TI, TO, 128>(p, inter, s);
}

template <typename TI>
int launch_append(const AppendParams& p, uint32_t type, uint32_t dim, bool inter, hipStream_t s) {
  return type == RLH_TYPE_F16 ? launch_append<TI, _Float16>(p, dim, inter, s) : launch_append<TI, __bf16>(p, dim, inter, s);
}

// Checks and enqueues an append; `positions` may be null.
int run_append(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_append_args* args, const uint32_t* positions,
               uint32_t* status, void* stream) {
  if (!args) return serve_error(RLH_EINVAL, "null argument");
  RLH_TRY(check_batch(kv, seqs, args->n_head));
  const uint32_t is = float_type_size(args->in_type);
  if (!is) return serve_error(RLH_EUNSUP, "in_type is not F32, F16 or BF16");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  const uint32_t D = kv->head_dim;
  const uint64_t qw = (uint64_t)args->n_head * D, kw = (uint64_t)kv->n_head_kv * D;
  RLH_TRY(check_rows("q", args->q, args->q_stride, qw, is));
  RLH_TRY(check_rows("k", args->k, args->k_stride, kw, is));
  RLH_TRY(check_rows("v", args->v, args->v_stride, kw, is));
  RLH_TRY(check_rows("q_out", args->q_out, args->q_out_stride, qw, 2));
  if (args->rot_dim % 16 || args->rot_dim > D)
    return serve_error(RLH_EINVAL, "rot_dim is not a multiple of 16 up to head_dim");
  if (args->rot_dim && !args->freqs) return serve_error(RLH_EINVAL, "freqs is null");
  if (!aligned(args->freqs, 8) || !aligned(args->q_norm, 16) || !aligned(args->k_norm, 16) || !aligned(status, 4))
    return serve_error(RLH_EINVAL, "freqs, q_norm, k_norm or status is misaligned");
  const uint64_t n = seqs->n_rows;
  const uint64_t ow = row_bytes_span(n, args->q_out_stride, qw, 2);
  if (overlap(args->q_out, ow, args->q, row_bytes_span(n, args->q_stride, qw, is)) ||
      overlap(args->q_out, ow, args->k, row_bytes_span(n, args->k_stride, kw, is)) ||
      overlap(args->q_out, ow, args->v, row_bytes_span(n, args->v_stride, kw, is)))
    return serve_error(RLH_EINVAL, "q_out overlaps q, k or v");
  if (overlaps_pool(*kv, args->q_out, ow) || overlaps_pool(*kv, args->q, row_bytes_span(n, args->q_stride, qw, is)) ||
      overlaps_pool(*kv, args->k, row_bytes_span(n, args->k_stride, kw, is)) ||
      overlaps_pool(*kv, args->v, row_bytes_span(n, args->v_stride, kw, is)))
    return serve_error(RLH_EINVAL, "the pool overlaps q, k, v or q_out");
  const Area q_start = area_q_start(*seqs), kv_len = area_kv_len(*seqs), table = area_table(*seqs, kv->page_size),
             q_norm = area("q_norm", args->q_norm, D * 4), k_norm = area("k_norm", args->k_norm, D * 4),
             freqs = area("freqs", args->rot_dim ? args->freqs : nullptr, args->rot_dim / 2 * 8),
             at = area("positions", positions, n * 4), st = area("status", status, 4), q_out{"q_out", args->q_out, n, args->q_out_stride * 2, qw * 2};
  for (const Area& written : {q_out, area("the pool", kv->k, pool_bytes(*kv)), area("the pool", kv->v, pool_bytes(*kv))})
    RLH_TRY(check_apart(written, {q_start, kv_len, table, q_norm, k_norm, freqs, at, st}));
  RLH_TRY(check_apart(st, {q_start, kv_len, table, q_norm, k_norm, freqs, at, Area{"q", args->q, n, args->q_stride * is, qw * is},
                           Area{"k", args->k, n, args->k_stride * is, kw * is},
                           Area{"v", args->v, n, args->v_stride * is, kw * is}}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("k pages", kv->k));
  RLH_TRY(dev("v pages", kv->v));
  RLH_TRY(dev("q_start", seqs->q_start));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("table", seqs->table));
  RLH_TRY(dev("q", args->q));
  RLH_TRY(dev("k", args->k));
  RLH_TRY(dev("v", args->v));
  RLH_TRY(dev("q_norm", args->q_norm));
  RLH_TRY(dev("k_norm", args->k_norm));
  if (args->rot_dim) RLH_TRY(dev("freqs", args->freqs));
  RLH_TRY(dev("positions", positions));
  RLH_TRY(dev("q_out", args->q_out));
  RLH_TRY(dev("status", status));
  AppendParams p{};
  p.b = Batch{seqs->n_seq, seqs->n_rows, seqs->max_q, seqs->max_kv, seqs->table_stride,
              seqs->q_start, seqs->kv_len, seqs->table};
  p.q = args->q;
  p.k = args->k;
  p.v = args->v;
  p.q_stride = args->q_stride;
  p.k_stride = args->k_stride;
  p.v_stride = args->v_stride;
  p.q_out_stride = args->q_out_stride;
  p.q_norm = args->q_norm;
  p.k_norm = args->k_norm;
  p.freqs = args->freqs;
  p.positions = positions;
  p.eps = args->eps;
  p.magnitude = args->magnitude;
  p.n_head = args->n_head;
  p.n_kv = kv->n_head_kv;
  p.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  p.n_pages = (uint32_t)kv->n_pages;
  p.rot_dim = args->rot_dim;
  p.q_out = args->q_out;
  p.pool_k = kv->k;
  p.pool_v = kv->v;
  p.status = status;
  const bool inter = args->interleaved != 0;
  if (args->in_type == RLH_TYPE_F32) return launch_append<float>(p, kv->type, D, inter, (hipStream_t)stream);
  if (args->in_type == RLH_TYPE_F16) return launch_append<_Float16>(p, kv->type, D, inter, (hipStream_t)stream);
  return launch_append<__bf16>(p, kv->type, D, inter, (hipStream_t)stream);
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

int rlh_rope_freqs(const rlh_rope* r, double* freqs, float* magnitude) {
  if (!r || !freqs || !magnitude) return serve_error(RLH_EINVAL, "null argument");
  if (r->rot_dim == 0 || r->rot_dim % 2 || r->rot_dim > 65536) return serve_error(RLH_EINVAL, "rot_dim is not a positive even number");
  if (!(r->theta > 1.0) || !isfinite(r->theta)) return serve_error(RLH_EINVAL, "theta is not above 1");
  if (r->scaling > RLH_ROPE_BANDS) return serve_error(RLH_EINVAL, "unknown rotary scaling");
  const double pi2 = 6.283185307179586;
  const bool bands = r->scaling == RLH_ROPE_BANDS;
  if (r->scaling != RLH_ROPE_PLAIN && (!(r->factor >= 1.0) || !isfinite(r->factor)))
    return serve_error(RLH_EINVAL, "factor is not at least 1");
  if (bands && (!(r->orig_ctx >= 1.0) || !isfinite(r->orig_ctx) || !(r->beta_slow > 0.0) ||
                !(r->beta_fast > r->beta_slow) || !isfinite(r->beta_fast)))
    return serve_error(RLH_EINVAL, "bands need orig_ctx >= 1 and beta_fast > beta_slow > 0");
  // the (real) index whose frequency turns t times over orig_ctx positions
  auto index_of = [&](double t) { return r->rot_dim * log(r->orig_ctx / (t * pi2)) / (2.0 * log(r->theta)); };
  const double lo = bands ? fmax(0.0, floor(index_of(r->beta_fast))) : 0.0;
  const double hi = bands ? fmin(r->rot_dim - 1.0, ceil(index_of(r->beta_slow))) : 0.0;
  for (uint32_t i = 0; i < r->rot_dim / 2; i++) {
    const double f = pow(r->theta, -2.0 * i / r->rot_dim);
    double slow = r->scaling == RLH_ROPE_LINEAR ? 1.0 : 0.0;
    if (bands) slow = fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 0.001)));
    freqs[i] = slow > 0.0 ? f * (1.0 - slow) + f / r->factor * slow : f;
  }
  *magnitude = bands ? (float)(0.1 * log(r->factor) + 1.0) : 1.0f;
  return RLH_OK;
}

int rlh_paged_append(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_append_args* args, uint32_t* status,
                     void* stream) {
  return run_append(kv, seqs, args, nullptr, status, stream);
}

int rlh_paged_append_at(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_append_args* args,
                        const uint32_t* positions, uint32_t* status, void* stream) {
  if (!positions && seqs && seqs->n_seq != 0 && seqs->n_rows != 0) return serve_error(RLH_EINVAL, "positions is null");
  if (!aligned(positions, 4)) return serve_error(RLH_EINVAL, "positions is not aligned to 4 bytes");
  return run_append(kv, seqs, args, positions, status, stream);
}

}  // extern "C"
