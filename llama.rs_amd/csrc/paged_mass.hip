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
  uint32_t stripes;     // blocks that share a KV head of a sequence
  uint64_t per_group;   // 2^36 / group, rounded up
};

// r / group: exact while r * group < 2^36 (a batch has up to 2^25 rows of all heads, a group up to 2^10).
__device__ __forceinline__ uint32_t of_group(const MassLaunch& L, uint32_t r) { return (uint32_t)(r * L.per_group >> 36); }

constexpr int kMassThreads = 256;

// Sum over the 16 lanes of a row, in every one of them.
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x128, 0xf, 0xf, true));  // row_ror 8
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x124, 0xf, 0xf, true));  // 4
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x122, 0xf, 0xf, true));  // 2
  x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x121, 0xf, 0xf, true));  // 1
  return x;
}

// What a weight needs to know of its row: exp(s - lse) is formed as 2^(s2 - lse2)
// * rest, where the log in units of log 2 is taken in two parts (one would put
// 2^-21 into every weight). The hardware's exponential has no values below 2^-126:
// such a weight is 0, which no sum with a larger one can tell.
struct MassRow {
  float lse2, rest, slope2;
  int32_t pos;  // of the row; below zero: it adds nothing
};
// The lse of row r of a KV head (minus infinity where there is none), and what follows from it.
__device__ __forceinline__ float mass_lse(const MassLaunch& L, const SeqView& v, uint32_t rows, uint32_t r, uint32_t h) {
  const AttnParams& a = L.a;
  const uint32_t i = of_group(L, r);
  return r < rows ? L.lse[(size_t)(v.q0 + i) * a.n_head + h * a.group + r - i * a.group] : -INFINITY;
}
__device__ __forceinline__ MassRow mass_row(const MassLaunch& L, const SeqView& v, uint32_t r, uint32_t h, bool biased, float lse) {
  const AttnParams& a = L.a;
  MassRow m{0.0f, 0.0f, 0.0f, -1};
  if (lse == -INFINITY) return m;
  const uint32_t i = of_group(L, r);
  if (biased && a.slopes) m.slope2 = a.slopes[h * a.group + r - i * a.group] * kLog2e;
  m.pos = (int32_t)(v.kv_len - v.q_len + i);
  m.lse2 = lse * kLog2e;
  const float rest = fmaf(lse, kLog2e, -m.lse2) + lse * kLog2eRest;
  m.rest = fabsf(m.lse2) < INFINITY ? __builtin_amdgcn_exp2f(-rest) : 1.0f;
  return m;
}
template <int MOD>
__device__ __forceinline__ float mass_weight(const Scoring& c, const MassRow& m, float dot, int32_t j) {
  const float x = MOD ? score<MOD>(c, dot, m.slope2, (float)(j - m.pos)) - m.lse2 : fmaf(dot, c.mul, -m.lse2);
  return __builtin_amdgcn_exp2f(x);
}

// The four positions from j0 on, whose places are m[0 .. 3]: x is added to what
// decays of `old` (of new positions, p0 and behind, nothing).
__device__ __forceinline__ void add_mass(float* m, f32x4_t old, f32x4_t x, float decay, int32_t j0, int32_t p0, int32_t n) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (decay != 0.0f && j0 + i < p0) x[i] = fmaf(decay, old[i], x[i]);
  if (j0 + 4 <= n) {
    *(f32x4_t*)m = x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (j0 + i < n) m[i] = x[i];
  }
}

// ---- single tokens and drafts ---------------------------------------------------------
// Up to 16 rows of a KV head: their queries stay in registers as the operand of
// an MFMA (16x16x32: positions down, rows across), and each wave streams K, 32
// positions at a time, one step ahead; a position's weights meet over the 16
// lanes that hold its rows. Every position has one owner: no atomics, no LDS.
// Bound by HBM: 61 tokens of 32 heads on 485 MB of keys and weights take 107 us
// (4.5 TB/s; without the step ahead, blocks of one step each: 135).
constexpr int kMassStep = 128;  // positions of a block's step, 32 per wave

template <typename T, int D, int MOD>
__global__ void __launch_bounds__(kMassThreads) k_mass_few(MassLaunch L) {
  constexpr int kSteps = D / 32;
  const AttnParams& a = L.a;
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t stripe = blockIdx.x % L.stripes, of = blockIdx.x / L.stripes, h = of % a.n_kv, s = of / a.n_kv;
  bool bad;
  SeqView v = load_seq(a.b, s, &bad);
  v.q0 = uniform(v.q0);
  v.q_len = uniform(v.q_len);
  v.kv_len = uniform(v.kv_len);
  if (bad && stripe == 0 && h == 0 && threadIdx.x == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
  if (!v.ok) return;
  const int32_t n = (int32_t)v.kv_len, p0 = n - (int32_t)v.q_len, hop = (int32_t)(L.stripes * kMassStep);
  int32_t p = (int32_t)(a.shared_len + stripe * kMassStep + wave * 32);
  if (p >= n) return;
  const uint32_t rows = v.q_len * a.group, prefix = a.prefix_len ? load_uniform(a.prefix_len, s) : 0;
  const uint32_t col = lane & 15, quad = lane >> 4;
  const uint32_t* table = a.b.table + (size_t)s * a.b.table_stride;
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  struct Step {
    u32x4_t k[2][kSteps];
    f32x4_t old;
    size_t at;    // of lanes with col < 2: where their four positions' masses lie
    uint32_t ok;  // which of the two groups of 16 positions exist
  };
  auto pages_of = [&](int32_t q, uint32_t (&page)[2]) {
#pragma unroll
    for (int u = 0; u < 2; u++) page[u] = q + 16 * u < n ? load_uniform(table, (uint32_t)(q + 16 * u) >> a.page_shift) : 0u;
  };
  auto fetch = [&](int32_t q, const uint32_t (&page)[2], Step& st) {
    st.ok = 0;
    size_t at[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const bool exists = q + 16 * u < n && page[u] < a.n_pages;
      if (q + 16 * u < n && !exists) raise(lane == 0 ? a.status : nullptr, RLH_SERVE_BAD_PAGE);
      st.ok |= exists ? 1u << u : 0u;
      at[u] = exists ? (((size_t)page[u] * a.n_kv + h) << a.page_shift) + ((uint32_t)(q + 16 * u) & page_mask) : 0;
      const T* kp = (const T*)a.pool_k + at[u] * D;
#pragma unroll
      for (int i = 0; i < kSteps; i++) st.k[u][i] = *(const RLH_GLOBAL u32x4_t*)(kp + (col * D + i * 32 + quad * 8));
    }
    st.at = (col ? at[1] : at[0]) + quad * 4;
    if (L.decay != 0.0f && col < 2 && q + 16 * (int32_t)col < n) st.old = *(const f32x4_t*)(L.mass + st.at);
  };
  uint32_t page[2];
  pages_of(p, page);
  const MassRow m = mass_row(L, v, col, h, MOD, mass_lse(L, v, rows, col, h));
  const RowSpan span = row_span(max(m.pos, 0), v.kv_len, a.window, prefix);
  // what every row sees, or none
  const RowSpan low = row_span(p0, v.kv_len, a.window, prefix), high = row_span(n - 1, v.kv_len, a.window, prefix);
  vec8<T> q[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; i++) {
    u32x4_t z = {0, 0, 0, 0};
    if (col < rows)
      z = *(const u32x4_t*)((const T*)a.q + (size_t)(v.q0 + col / a.group) * a.q_stride +
                            (size_t)(h * a.group + col % a.group) * D + i * 32 + quad * 8);
    q[i] = __builtin_bit_cast(vec8<T>, z ^ L.sc.flip);
  }
  Step cur, next;
  fetch(p, page, cur);
  pages_of(p + hop, page);
  for (; p < n; p += hop) {
    if (p + hop < n) {
      fetch(p + hop, page, next);
      pages_of(p + 2 * hop, page);
    }
    float sum[8] = {};
    if ((p < high.hi && p + 32 > low.lo) || p < low.prefix) {
      const bool full = (p >= high.lo && p + 32 <= low.hi) || p + 32 <= low.prefix;
      f32x4_t sc[2] = {f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < kSteps; i++)
#pragma unroll
        for (int u = 0; u < 2; u++) sc[u] = mfma16(__builtin_bit_cast(vec8<T>, cur.k[u][i]), q[i], sc[u]);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int32_t j = p + (i / 4) * 16 + (int32_t)quad * 4 + i % 4;
        const float w = mass_weight<MOD>(L.sc, m, sc[i / 4][i % 4], j) * m.rest;
        sum[i] = ((m.pos >= 0) & (full | row_sees(span, j))) ? w : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) sum[i] = row_sum(sum[i]);
    }
    // lane (quad, u) has the four positions of quad `quad` of group u
    if (col < 2 && (cur.ok >> col & 1)) {
      const int32_t j0 = p + (int32_t)(col * 16 + quad * 4);
      add_mass(L.mass + cur.at, cur.old, col ? f32x4_t{sum[4], sum[5], sum[6], sum[7]} : f32x4_t{sum[0], sum[1], sum[2], sum[3]},
               L.decay, j0, p0, n);
    }
    cur = next;
  }
}

// ---- many rows ------------------------------------------------------------------------
// A wave keeps K of 32 positions of one KV head in registers; the block's rows
// pass by in LDS, 64 at a time and the next ones on their way, as the other
// operand of 32x32x16 MFMAs (positions down, rows across). Each score becomes its
// weight and joins one register per lane and position; the lanes of a position
// meet once at the end. Four blocks run on a CU and hide each other's starts (64
// positions a wave and two blocks: 82 us instead of 59 for 3 sequences of 20000
// positions and 256 rows). Bound by HBM up to 64 rows (28 us for 32 rows, 4.5 TB/s),
// then by exponentials and products in turn (1024 rows: 592 TFLOP/s).
constexpr int kMassRows = 64;
constexpr int kMassTile = 128;  // positions of a block

template <typename T, int D, int MOD>
__global__ void __launch_bounds__(kMassThreads, 4) k_mass_many(MassLaunch L) {
  constexpr int kSteps = D / 16;
  constexpr int kLanes = D / 8;           // lanes of a row in a copy
  constexpr int kBuf = kMassRows * D * 2;
  constexpr int kCopies = kBuf / 1024 / (kMassThreads / 64);
  __shared__ __align__(16) uint8_t qs[2 * kBuf];
  __shared__ MassRow infos[2][kMassRows];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(RLH_LDS uint8_t*)qs;
  const AttnParams& a = L.a;
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, t = threadIdx.x;
  const uint32_t stripe = blockIdx.x % L.stripes, of = blockIdx.x / L.stripes, h = of % a.n_kv, s = of / a.n_kv;
  bool bad;
  SeqView v = load_seq(a.b, s, &bad);
  v.q0 = uniform(v.q0);
  v.q_len = uniform(v.q_len);
  v.kv_len = uniform(v.kv_len);
  if (bad && stripe == 0 && h == 0 && t == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
  if (!v.ok) return;
  const uint32_t rows = v.q_len * a.group, prefix = a.prefix_len ? load_uniform(a.prefix_len, s) : 0;
  const int32_t n = (int32_t)v.kv_len, p0 = n - (int32_t)v.q_len;
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t* table = a.b.table + (size_t)s * a.b.table_stride;
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  // rows c0 .. into buffer `buf` (behind the last one that one again: it adds nothing)
  auto stage = [&](uint32_t c0, uint32_t buf) {
#pragma unroll
    for (int i = 0; i < kCopies; i++) {
      const uint32_t piece = wave * kCopies + i, r = piece * (64 / kLanes) + lane / kLanes, rr = min(c0 + r, rows - 1);
      const uint32_t at = of_group(L, rr);
      const T* row = (const T*)a.q + (size_t)(v.q0 + at) * a.q_stride + (size_t)(h * a.group + rr - at * a.group) * D;
      copy_to_lds(row + ((lane % kLanes) ^ swizzle<D>(r)) * 8, uniform(lds0 + buf * kBuf + piece * 1024));
    }
  };
  // what rows r .. end - 1 see of positions q .. q_end - 1: 0 nothing, 2 each row all, else 1
  auto sees = [&](uint32_t r, uint32_t end, int32_t q, int32_t q_end) -> int {
    const RowSpan low = row_span(p0 + (int32_t)of_group(L, r), v.kv_len, a.window, prefix);
    const RowSpan high = row_span(p0 + (int32_t)of_group(L, end - 1), v.kv_len, a.window, prefix);
    if (!((q < high.hi && q_end > low.lo) || q < low.prefix)) return 0;
    return (q >= high.lo && q_end <= low.hi) || q_end <= low.prefix ? 2 : 1;
  };
  for (int32_t b0 = (int32_t)(a.shared_len + stripe * kMassTile); b0 < n; b0 += (int32_t)(L.stripes * kMassTile)) {
    const int32_t p = b0 + (int32_t)wave * 32, b1 = min(b0 + kMassTile, n);
    // the rows from c on that see any of the block's positions
    auto next_rows = [&](uint32_t c) {
      while (c < rows && sees(c, min(c + kMassRows, rows), b0, b1) == 0) c += kMassRows;
      return uniform(min(c, rows));
    };
    uint32_t c0 = next_rows(0), buf = 0;
    __syncthreads();  // every wave is done with what lies in LDS
    float lse = -INFINITY;
    if (c0 < rows) {
      stage(c0, 0);
      if (t < kMassRows) lse = mass_lse(L, v, rows, c0 + t, h);
    }
    // pages of the wave's two groups of 16 positions
    uint32_t page[2], ok = 0;
    size_t at[2];
#pragma unroll
    for (int u = 0; u < 2; u++) page[u] = p + 16 * u < n ? load_uniform(table, (uint32_t)(p + 16 * u) >> a.page_shift) : 0u;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const bool live = p + 16 * u < n, exists = live && page[u] < a.n_pages;
      ok |= (exists ? 1u << u : 0u) | (live && !exists ? 4u : 0u);
      at[u] = exists ? (((size_t)page[u] * a.n_kv + h) << a.page_shift) + ((uint32_t)(p + 16 * u) & page_mask) : 0;
    }
    if (ok & 4) raise(lane == 0 ? a.status : nullptr, RLH_SERVE_BAD_PAGE);
    vec8<T> k[kSteps];  // (negated where the scale is: the rows come unchanged)
    {
      const T* kp = (const T*)a.pool_k + ((col & 16 ? at[1] : at[0]) + (col & 15)) * D + half * 8;
#pragma unroll
      for (int i = 0; i < kSteps; i++) k[i] = __builtin_bit_cast(vec8<T>, *(const u32x4_t*)(kp + i * 16) ^ L.sc.flip);
    }
    if (t < kMassRows) infos[0][t] = mass_row(L, v, c0 + t, h, MOD, lse);
    float sum[16] = {};
    while (c0 < rows) {
      const uint32_t c1 = min(c0 + kMassRows, rows), c2 = next_rows(c0 + kMassRows);
      wait_vmcnt<0>();  // this wave's rows have landed
      __syncthreads();  // ... everyone's; every wave is done with the other buffer
      if (c2 < rows) {
        if (t < kMassRows) lse = mass_lse(L, v, rows, c2 + t, h);
        stage(c2, buf ^ 1);
      }
      const uint8_t* q0 = qs + buf * kBuf;
      const int whole = sees(c0, c1, p, p + 32);
      for (uint32_t r0 = c0; r0 < c1; r0 += 32) {
        const int see = whole == 1 ? sees(r0, min(r0 + 32, rows), p, p + 32) : whole;
        if (see == 0) continue;
        const uint32_t r = r0 - c0 + col;
        vec8<T> q[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; i++) q[i] = *(const vec8<T>*)(q0 + r * D * 2 + ((2 * i + half) ^ swizzle<D>(r)) * 16);
        const MassRow m = infos[buf][r];
        f32x16_t sc;
#pragma unroll
        for (int e = 0; e < 16; e++) sc[e] = 0.0f;
        __builtin_amdgcn_sched_barrier(0);  // (all reads before the first product: one takes some 250 cycles)
#pragma unroll
        for (int i = 0; i < kSteps; i++) sc = mfma32(k[i], q[i], sc);
        // the lane's first position (opaque, so that 16 of them are not kept in registers)
        int32_t j0 = p + (int32_t)half * 4;
        asm volatile("" : "+v"(j0));
#pragma unroll
        for (int i = 0; i < 16; i++)
          sc[i] = mass_weight<MOD>(L.sc, m, sc[i], j0 + i / 4 * 8 + i % 4);
        if (see != 2 || __ballot(m.pos < 0)) {
          const RowSpan span = row_span(max(m.pos, 0), v.kv_len, a.window, prefix);
          const bool counts = m.pos >= 0;
          const int32_t lo = counts ? span.lo - j0 : 0x7fffffff, hi = span.hi - j0, pre = counts ? span.prefix - j0 : -0x7fffffff;
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int32_t d = i / 4 * 8 + i % 4;
            sc[i] = (((d >= lo) & (d < hi)) | (d < pre)) ? sc[i] : 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) sum[i] = fmaf(sc[i], m.rest, sum[i]);
      }
      if (t < kMassRows && c2 < rows) infos[buf ^ 1][t] = mass_row(L, v, c2 + t, h, MOD, lse);
      c0 = c2;
      buf ^= 1;
    }
    // Lane (col, half) has positions 8 g + 4 half + 0..3; lane col = g writes its four.
    f32x4_t mine = {0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < 4; g++) {
      f32x4_t x;
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = sum_across_16(row_sum(sum[g * 4 + i]));
      if (col == (uint32_t)g) mine = x;
    }
    if (col < 4 && (ok >> (col >> 1) & 1)) {
      const int32_t j0 = p + (int32_t)(col * 8 + half * 4);
      float* dst = L.mass + (col >> 1 ? at[1] : at[0]) + (col & 1) * 8 + half * 4;
      const f32x4_t old = L.decay != 0.0f && j0 < p0 ? *(const f32x4_t*)dst : f32x4_t{0, 0, 0, 0};
      add_mass(dst, old, mine, L.decay, j0, p0, n);
    }
  }
}

template <typename T, int D, int MOD>
int launch_mass(const MassLaunch& L, bool few, hipStream_t s) {
  return enqueue("rlh_paged_mass", few ? k_mass_few<T, D, MOD> : k_mass_many<T, D, MOD>, dim3(L.a.b.n_seq * L.a.n_kv * L.stripes),
                 kMassThreads, 0, s, L);
}

template <typename T, int D>
int launch_mass(const MassLaunch& L, int mod, bool few, hipStream_t s) {
  return mod == kPlain ? launch_mass<T, D, kPlain>(L, few, s)
         : mod == kMod ? launch_mass<T, D, kMod>(L, few, s) : launch_mass<T, D, kWideCap>(L, few, s);
}

template <typename T>
int launch_mass(const MassLaunch& L, uint32_t dim, int mod, bool few, hipStream_t s) {
  return dim == 64 ? launch_mass<T, 64>(L, mod, few, s) : launch_mass<T, 128>(L, mod, few, s);
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
  L.a.window = args->window & ~RLH_WINDOW_DRAFTS;
  L.a.shared_len = args->shared_len;
  L.per_group = ((1ull << 36) + L.a.group - 1) / L.a.group;
  L.lse = lse;
  L.mass = mass;
  L.decay = decay;
  if (seqs->max_kv <= args->shared_len) return RLH_OK;
  // Blocks share a sequence's positions, no more of them than there are steps: few
  // rows go on from step to step, sixteen blocks to a CU in all; many have a step each.
  const bool few = (uint64_t)seqs->max_q * L.a.group <= 16;
  const uint32_t step = few ? kMassStep : kMassTile, most = (seqs->max_kv - args->shared_len + step - 1) / step;
  L.stripes = std::min(most, std::max(1u, (few ? 4096u : 65536u) / (seqs->n_seq * kv->n_head_kv)));
  int mod;
  L.sc = scoring_of(*args, &mod);
  if (kv->type == RLH_TYPE_F16) return launch_mass<_Float16>(L, kv->head_dim, mod, few, (hipStream_t)stream);
  return launch_mass<__bf16>(L, kv->head_dim, mod, few, (hipStream_t)stream);
}

}  // extern "C"
