// paged_mass.hip — the attention weight that each cached position gathers.
#include "../../include/rlh_cache.h"
#include "paged_attn.h"

namespace rlh {
namespace {

struct MassLaunch {
  AttnParams a;  // its out, shared table and parts of a workspace are not used
  Scoring sc;
  const float* lse;
  float* mass;
  float decay;
  uint32_t stripes;  // blocks that share a KV head of a sequence
};

constexpr int kMassThreads = 256;
constexpr int kMassStep = 128;  // positions of a block's step, 32 per wave

// Sum over the 16 lanes of a row, in every one of them.
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x128, 0xf, 0xf, true));  // row_ror 8
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x124, 0xf, 0xf, true));  // 4
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x122, 0xf, 0xf, true));  // 2
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x121, 0xf, 0xf, true));  // 1
  return x;
}

// A wave takes 32 positions of one KV head and all rows that see them, 16 at a
// time: K goes straight into MFMA operands (positions down, rows across), a
// score becomes its weight with the row's known sum, and the weights of a
// position add up in one register per lane, over all rows; the lanes of a
// position meet once at the end. Every position has one owner: no atomics.
template <typename T, int D, int MOD>
__global__ void __launch_bounds__(kMassThreads) k_paged_mass(MassLaunch L) {
  constexpr int kSteps = D / 32;
  const AttnParams& a = L.a;
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t stripe = blockIdx.x % L.stripes, of = blockIdx.x / L.stripes, h = of % a.n_kv, s = of / a.n_kv;
  bool bad;
  const SeqView v = load_seq(a.b, s, &bad);
  if (bad && stripe == 0 && h == 0 && threadIdx.x == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
  if (!v.ok) return;
  const uint32_t rows = v.q_len * a.group, prefix = a.prefix_len ? a.prefix_len[s] : 0;
  const int32_t n = (int32_t)v.kv_len, p0 = n - (int32_t)v.q_len;
  const uint32_t col = lane & 15, quad = lane >> 4;
  const uint32_t* table = a.b.table + (size_t)s * a.b.table_stride;
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  for (int32_t p = (int32_t)(a.shared_len + stripe * kMassStep + wave * 32); p < n; p += (int32_t)(L.stripes * kMassStep)) {
    u32x4_t kr[2][kSteps];
    size_t at[2];
    uint32_t ok = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int32_t pu = p + 16 * u;
      uint32_t page = pu < n ? load_uniform(table, (uint32_t)pu >> a.page_shift) : 0u;
      bool exists = pu < n;
      if (exists && page >= a.n_pages) {
        raise(lane == 0 ? a.status : nullptr, RLH_SERVE_BAD_PAGE);
        exists = false;
      }
      if (!exists) page = 0;
      ok |= exists ? 1u << u : 0u;
      at[u] = (((size_t)page * a.n_kv + h) << a.page_shift) + (exists ? (uint32_t)pu & page_mask : 0);
      const T* kp = (const T*)a.pool_k + at[u] * D;
#pragma unroll
      for (int i = 0; i < kSteps; i++) kr[u][i] = *(const RLH_GLOBAL u32x4_t*)(kp + (col * D + i * 32 + quad * 8));
    }
    if (!ok) continue;
    float sum[8] = {};
    for (uint32_t r0 = 0; r0 < rows; r0 += 16) {
      const int32_t pos_a = p0 + (int32_t)(r0 / a.group), pos_b = p0 + (int32_t)(min(r0 + 15, rows - 1) / a.group);
      const RowSpan low = row_span(pos_a, v.kv_len, a.window, prefix), high = row_span(pos_b, v.kv_len, a.window, prefix);
      // whether any row sees any of the positions; whether all see all
      if (!((p < high.hi && p + 32 > low.lo) || p < low.prefix)) continue;
      const bool full = (p >= high.lo && p + 32 <= low.hi) || p + 32 <= low.prefix;
      const uint32_t rr = r0 + col;
      const bool active = rr < rows;
      const uint32_t row = v.q0 + (active ? rr / a.group : 0), head = h * a.group + (active ? rr % a.group : 0);
      const int32_t pos = p0 + (int32_t)(row - v.q0);
      const RowSpan span = row_span(pos, v.kv_len, a.window, prefix);
      const float slope2 = MOD && a.slopes ? a.slopes[head] * kLog2e : 0.0f;
      // log2 of the row's sum in two parts: one would put 2^-21 into every weight
      float lse = active ? L.lse[(size_t)row * a.n_head + head] : -INFINITY;
      const bool counts = lse != -INFINITY;
      if (!counts) lse = 0.0f;
      const float lse2 = lse * kLog2e;
      const float rest = fmaf(lse, kLog2e, -lse2) + lse * kLog2eRest;
      const float f = fabsf(lse2) < INFINITY ? __builtin_amdgcn_exp2f(-rest) : 1.0f;
      f32x4_t sc[2] = {f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        u32x4_t q = {0, 0, 0, 0};
        if (active) q = *(const u32x4_t*)((const T*)a.q + (size_t)row * a.q_stride + (size_t)head * D + i * 32 + quad * 8);
        const vec8<T> qv = __builtin_bit_cast(vec8<T>, q ^ L.sc.flip);
#pragma unroll
        for (int u = 0; u < 2; u++) sc[u] = mfma16(__builtin_bit_cast(vec8<T>, kr[u][i]), qv, sc[u]);
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int32_t j = p + (i / 4) * 16 + (int32_t)quad * 4 + i % 4;
        const float d = sc[i / 4][i % 4];
        const float x = MOD ? score<MOD>(L.sc, d, slope2, (float)(j - pos)) - lse2 : fmaf(d, L.sc.mul, -lse2);
        const float w = __builtin_amdgcn_exp2f(x);
        if (counts & (full | row_sees(span, j))) sum[i] = fmaf(w, f, sum[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = row_sum(sum[i]);
    // lane (quad, u) has the four positions of quad `quad` of group u
    if (col >= 2 || !(ok >> col & 1)) continue;
    const int32_t j0 = p + (int32_t)(col * 16 + quad * 4);
    float* m = L.mass + (col ? at[1] : at[0]) + quad * 4;
    f32x4_t x;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = col ? sum[4 + i] : sum[i];
    if (j0 + 4 <= n) {
      if (L.decay != 0.0f) {
        const f32x4_t old = *(const f32x4_t*)m;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (j0 + i < p0) x[i] = fmaf(L.decay, old[i], x[i]);
      }
      *(f32x4_t*)m = x;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (j0 + i < n) m[i] = L.decay != 0.0f && j0 + i < p0 ? fmaf(L.decay, m[i], x[i]) : x[i];
    }
  }
}

template <typename T, int D>
int launch_mass(const MassLaunch& L, int mod, hipStream_t s) {
  const dim3 grid(L.a.b.n_seq * L.a.n_kv * L.stripes);
  const auto kernel = mod == kPlain ? k_paged_mass<T, D, kPlain>
                      : mod == kMod ? k_paged_mass<T, D, kMod> : k_paged_mass<T, D, kWideCap>;
  return enqueue("rlh_paged_mass", kernel, grid, kMassThreads, 0, s, L);
}

template <typename T>
int launch_mass(const MassLaunch& L, uint32_t dim, int mod, hipStream_t s) {
  return dim == 64 ? launch_mass<T, 64>(L, mod, s) : launch_mass<T, 128>(L, mod, s);
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

int rlh_paged_mass(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, const float* lse,
                   float decay, float* mass, uint32_t* status, void* stream) {
  RLH_TRY(check_scores(kv, seqs, args));
  if (!(decay >= 0.0f) || !isfinite(decay)) return serve_error(RLH_EINVAL, "decay is negative or not finite");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  if (!lse || !aligned(lse, 4)) return serve_error(RLH_EINVAL, "lse is null or not aligned to 4 bytes");
  if (!mass || !aligned(mass, 16)) return serve_error(RLH_EINVAL, "mass is null or not aligned to 16 bytes");
  if (!aligned(status, 4)) return serve_error(RLH_EINVAL, "status is not aligned to 4 bytes");
  const uint64_t n = seqs->n_rows, w = (uint64_t)args->n_head * kv->head_dim;
  const Area q_start = area_q_start(*seqs), kv_len = area_kv_len(*seqs), table = area_table(*seqs, kv->page_size),
             slopes = area("slopes", args->slopes, args->n_head * 4ull),
             prefix_len = area("prefix_len", args->prefix_len, seqs->n_seq * 4ull),
             q{"q", args->q, n, args->q_stride * 2, w * 2}, sums = area("lse", lse, n * args->n_head * 4),
             keys = area("the pool", kv->k, pool_bytes(*kv)), values = area("the pool", kv->v, pool_bytes(*kv)),
             out = area("mass", mass, kv->n_pages * kv->n_head_kv * kv->page_size * 4), st = area("status", status, 4);
  RLH_TRY(check_apart(out, {q_start, kv_len, table, slopes, prefix_len, q, sums, keys, values, st}));
  RLH_TRY(check_apart(st, {q_start, kv_len, table, slopes, prefix_len, q, sums, keys, values}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("k pages", kv->k));
  RLH_TRY(dev("q_start", seqs->q_start));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("table", seqs->table));
  RLH_TRY(dev("q", args->q));
  RLH_TRY(dev("slopes", args->slopes));
  RLH_TRY(dev("prefix_len", args->prefix_len));
  RLH_TRY(dev("lse", lse));
  RLH_TRY(dev("mass", mass));
  RLH_TRY(dev("status", status));
  MassLaunch L{};
  L.a.b = Batch{seqs->n_seq, seqs->n_rows, seqs->max_q, seqs->max_kv, seqs->table_stride,
                seqs->q_start, seqs->kv_len, seqs->table};
  L.a.q = args->q;
  L.a.pool_k = kv->k;
  L.a.q_stride = args->q_stride;
  L.a.slopes = args->slopes;
  L.a.prefix_len = args->prefix_len;
  L.a.status = status;
  L.a.n_head = args->n_head;
  L.a.n_kv = kv->n_head_kv;
  L.a.group = args->n_head / kv->n_head_kv;
  L.a.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  L.a.n_pages = (uint32_t)kv->n_pages;
  L.a.window = args->window;
  L.a.shared_len = args->shared_len;
  L.lse = lse;
  L.mass = mass;
  L.decay = decay;
  if (seqs->max_kv <= args->shared_len) return RLH_OK;
  const uint32_t most = (seqs->max_kv - args->shared_len + kMassStep - 1) / kMassStep;
  L.stripes = std::min(most, std::max(1u, 65536u / (seqs->n_seq * kv->n_head_kv)));
  int mod;
  L.sc = scoring_of(*args, &mod);
  if (kv->type == RLH_TYPE_F16) return launch_mass<_Float16>(L, kv->head_dim, mod, (hipStream_t)stream);
  return launch_mass<__bf16>(L, kv->head_dim, mod, (hipStream_t)stream);
}

}  // extern "C"
