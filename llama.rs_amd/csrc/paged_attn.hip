// paged_attn.hip — attention of a ragged batch over the paged cache.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "paged_device.h"
#include "rlh_device.h"
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
  uint32_t n_head, n_kv, group, page_shift, n_pages, window, shared_len;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kSmallRows = 16;    // rows of a KV head that the small kernel takes (the width of its MFMA)
constexpr int kTileWaves = 8;
constexpr int kTileRows = 32 * kTileWaves;  // rows of a tile of the tiled kernel
constexpr int kTileKv = 64;       // positions of its steps
// The maximum that probabilities are relative to is only moved when the
// running maximum has grown by more than 8 (in units of log 2): until then
// they stay below 2^8 times the factor below, which f16 holds.
constexpr float kSlack = 8.0f;
// Probabilities of f16 are formed 2^7 larger, just below f16's largest, in the
// products with V and in their sums alike: what lies below 2^-14 of the maximum
// would lose bits as f16 and vanish below 2^-25, though the sum counts it (20000
// positions 17.5 below one: all of their share of the result). bf16 has f32's exponents.
template <typename T>
constexpr float kLift = __is_same(T, _Float16) ? 7.0f : 0.0f;

#define RLH_CONST __attribute__((address_space(4)))
#define RLH_LDS_PTR(T) __attribute__((address_space(3))) T

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// A value every lane of the wave has.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t load_uniform(const uint32_t* p, uint32_t i) {
  return *((const RLH_CONST uint32_t*)p + uniform(i));
}

__device__ __forceinline__ float max_across_32(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_across_16(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across_32(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_across_16(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma16(vec8<_Float16> a, vec8<_Float16> b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(vec8<__bf16> a, vec8<__bf16> b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma32(vec8<_Float16> a, vec8<_Float16> b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma32(vec8<__bf16> a, vec8<__bf16> b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Columns of V as an MFMA operand: a group of 16 lanes names four rows of 16
// values (lane t: row t / 4, values 4 (t % 4) .. + 3) and gets the transpose,
// lane t the four rows' value t. Two of them make an operand's eight.
template <typename T>
__device__ __forceinline__ vec8<T> read_columns(const uint8_t RLH_LDS* a, const uint8_t RLH_LDS* b) {
  const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RLH_LDS_PTR(s16x4_t)*)a);
  const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((RLH_LDS_PTR(s16x4_t)*)b);
  return __builtin_bit_cast(vec8<T>, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Whether any of eight halves is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool any_special(u32x4_t x) {
  constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
  bool r = false;
#pragma unroll
  for (int i = 0; i < 4; i++) r |= (x[i] & e) == e || (x[i] >> 16 & e) == e;
  return r;
}

// Element i (the same in every lane) of the vector that lane `src` holds.
template <typename T>
__device__ __forceinline__ float element(vec8<T> v, uint32_t i, int src) {
  const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  const uint32_t x = i < 4 ? (i < 2 ? w[0] : w[1]) : (i < 6 ? w[2] : w[3]);
  const uint32_t y = __shfl(x, src);
  return (float)__builtin_bit_cast(T, (uint16_t)(i & 1 ? y >> 16 : y));
}

// Copies 16 bytes per lane to LDS from `dst` on (the same in every lane), in
// lane order, without registers; counted by vmcnt. Written out so that the
// compiler does not make every later read by columns wait for it: the step's
// own wait and barrier order them. (m0 is reserved, which the compiler warns
// of; named all the same, it orders this against the compiler's own uses.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(dst) : "memory", "m0");
}
#pragma clang diagnostic pop

// Scores in units of log 2. Without cap and bias they are dot * mul, and the
// product is only formed in the exponential's argument (mul > 0: the largest
// dot has the largest score).
struct Scoring {
  float mul;              // |scale| * log2(e), or with a cap 2 scale / cap * log2(e)
  float cap2;             // softcap * log2(e)
  uint32_t flip;          // sign bits of two halves: q is negated where scale < 0
  bool capped, biased;
};
// What the kernels' variants do to a score: nothing, cap and bias, or the same
// with a cap above kNarrowCap (a variant of its own: the wide form beside the
// other in one kernel made prompts with a bias 3 % slower).
enum { kPlain = 0, kMod = 1, kWideCap = 2 };

// Up to this cap a score may be off by 2^-23 of the cap (a probability by
// 2^-17 of itself); above, tanh's own size counts.
constexpr float kNarrowCap = 64.0f;
// Larger caps are taken as this one, which changes no score below 2^88 in f32.
constexpr float kMostCap = 0x1p100f;

// tanh(y) = 1 - 2 / (exp(2 y) + 1): off by 2^-23 of the cap, at any y
__device__ __forceinline__ float capped(const Scoring& c, float dot) {
  return fmaf(-2.0f * c.cap2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * c.mul) + 1.0f), c.cap2);
}
// Below |y| = 1/4 by the series y (1 - y^2 / 3 + 2 y^4 / 15 - 17 y^6 / 315 + 62
// y^8 / 2835), off by 2^-26 of itself; x = dot * mul is y times 2 log2(e). The
// products with the cap then cancel: a cap of any size leaves small scores as they are.
__device__ __forceinline__ float capped_wide(const Scoring& c, float dot) {
  constexpr float a = 0.34657359f, a2 = a * a;  // ln(2) / 2
  const float x = dot * c.mul, z = x * x;
  float p = a2 * a2 * a2 * a2 * 62.0f / 2835.0f;
  p = fmaf(p, z, -a2 * a2 * a2 * 17.0f / 315.0f);
  p = fmaf(p, z, a2 * a2 * 2.0f / 15.0f);
  p = fmaf(p, z, -a2 / 3.0f);
  p = fmaf(p, z, 1.0f);
  return fabsf(x) < 0.72134752f ? x * (c.cap2 * a) * p : capped(c, dot);
}
template <int MOD>
__device__ __forceinline__ float score(const Scoring& c, float dot, float slope2, float away) {
  const float x = MOD == kWideCap ? capped_wide(c, dot) : c.capped ? capped(c, dot) : dot * c.mul;
  return c.biased ? fmaf(slope2, away, x) : x;
}

// What the partial results of one row look like: m, l and the D sums, by
// source: prefix parts, then the parts of the sequence's own positions.
struct Workspace {
  float* prefix_o;   // [prefix_parts][n_rows * n_head][D]
  float* prefix_ml;  // [prefix_parts][n_rows * n_head][2]
  float* tile_o;     // [tile_parts][n_rows * n_head][D]
  float* tile_ml;
  float* item_o;     // [items * n_kv][16][D]
  float* item_ml;    // [items * n_kv][16][2]
  uint32_t* plan;    // [n_seq][2]: first item, items
  uint32_t* tiles;   // [n_seq][2]: first tile, tiles (where `planned`)
};

struct Sizes {
  uint32_t items;         // at most, of the small kernel (per KV head)
  uint32_t item_goal;     // items that its work is divided into (and one more per sequence)
  uint32_t tiles;         // at most, of the tiled kernel (per KV head)
  uint32_t tile_parts;    // parts of the positions of a tile
  uint32_t prefix_tiles;  // tiles over all rows
  uint32_t prefix_parts;  // of all but the last of them
  uint32_t last_parts;    // of the last, which may have fewer rows
  uint32_t small_rows;    // sequences of up to so many rows of a KV head go to the small kernel
  bool small, tiled, merge;
  bool whole;             // the small kernel's sequences are not divided
  bool planned;           // a launch before found where each sequence's items and tiles begin
  bool merge_small;       // only its sequences have parts to join
  uint32_t merge_rows;    // then: blocks per sequence and KV head
};

// Blocks of a KV head for the shared prefix.
__host__ __device__ inline uint32_t prefix_blocks(const Sizes& n) {
  return n.prefix_tiles ? (n.prefix_tiles - 1) * n.prefix_parts + n.last_parts : 0;
}

struct Launch {
  AttnParams a;
  Scoring sc;
  Workspace ws;
  Sizes n;
};

struct SeqSpan {
  SeqView v;
  uint32_t rows;      // of a KV head: new rows times heads per KV head
  int32_t p0;         // position of the first new row
  int32_t begin, end; // positions that any of its rows sees (own ones: from shared_len)
  uint32_t prefix;
};

__device__ __forceinline__ SeqSpan seq_span(const AttnParams& a, uint32_t s, bool* bad) {
  SeqSpan r;
  r.v = load_seq(a.b, s, bad);
  r.rows = r.v.ok ? r.v.q_len * a.group : 0;
  r.p0 = (int32_t)(r.v.kv_len - r.v.q_len);
  r.prefix = a.prefix_len ? a.prefix_len[s] : 0;
  r.begin = r.end = 0;
  if (r.v.ok) {
    const int32_t b = span_begin(row_span(r.p0, r.v.kv_len, a.window, r.prefix));
    r.begin = (b > (int32_t)a.shared_len ? b : (int32_t)a.shared_len) & ~15;
    r.end = span_end(row_span((int32_t)r.v.kv_len - 1, r.v.kv_len, a.window, r.prefix));
  }
  return r;
}

// x moved between lanes by a DPP control; 0 where none comes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
// Inclusive sum over the wave in lane order.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += dpp0<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += dpp0<0x112, 0xf>(x);
  x += dpp0<0x114, 0xf>(x);
  x += dpp0<0x118, 0xf>(x);
  x += dpp0<0x142, 0xa>(x);  // row_bcast 15, 31
  x += dpp0<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t x, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// Finds item `item` of a list in which sequence s has parts(s) items, one
// after the other: every wave for itself, 64 sequences at a time (no
// barriers). False if the list ends before it.
struct Found {
  uint32_t s, first, n;  // the sequence, its first item, its items
};
template <typename F>
__device__ __forceinline__ bool find_item(uint32_t n_seq, uint32_t item, F parts, Found* f) {
  uint32_t base = 0;
  for (uint32_t s0 = 0; s0 < n_seq; s0 += 64) {
    const uint32_t s = s0 + (threadIdx.x & 63);
    const uint32_t n = s < n_seq ? parts(s) : 0;
    const uint32_t upto = base + wave_scan(n);
    const uint64_t hit = __ballot(upto > item);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      f->s = s0 + (uint32_t)l;
      f->n = lane_value(n, l);
      f->first = lane_value(upto, l) - f->n;
      return true;
    }
    base = lane_value(upto, 63);
  }
  return false;
}

// The same in a list that k_attn_plan left.
__device__ __forceinline__ bool find_planned(const uint32_t* plan, uint32_t n_seq, uint32_t item, Found* f) {
  const uint32_t n = count_upto(plan, 2, n_seq, item);
  if (n == 0) return false;
  f->s = n - 1;
  f->first = load_uniform(plan, 2 * f->s);
  f->n = load_uniform(plan, 2 * f->s + 1);
  return item < f->first + f->n;
}

// Steps of a block of W waves over the positions of sequence s, and whether it
// is one of few rows.
template <int W>
__device__ __forceinline__ uint32_t small_steps(const AttnParams& a, uint32_t s, bool* bad, bool* mine) {
  const SeqSpan q = seq_span(a, s, bad);
  *mine = q.rows != 0 && q.rows <= kSmallRows;
  return *mine && q.end > q.begin ? (uint32_t)(q.end - q.begin + 32 * W - 1) / (32 * W) : 0;
}

// ---- few rows: single tokens and drafts -----------------------------------------
// A block takes one KV head of one sequence (up to 16 rows) and a part of
// its positions; each wave streams 32 positions at a time on its own: K
// straight into MFMA operands (16x16x32: positions down, rows across), V
// through the wave's LDS rows to be read by columns. Scores come out with a
// row per lane column, so the running maximum and the sum are one register per
// lane, and the probabilities are already the next product's operand if V's
// rows are taken in the order that the lanes hold them: 4 (lane / 16) + i, and
// 16 more. Probabilities are rounded to the pool's type for that product (off
// by half a step of each; the sum takes them unrounded), all else is f32.
// Bound by HBM: 61 tokens of 32 heads on 940 MB of pages take 166 us (5.7
// TB/s; a copy of 2 GiB moves 5.1), 3 of 64 heads on 459 MB 90 us. The
// positions are divided so that the parts are of one length, 768 blocks of them
// (of the two or three that a CU runs at once); a single short sequence costs the chain of loads from its start to its
// pages (6 us) and the second launch that joins the parts (4 us).
template <int D, int W>
constexpr uint32_t kSmallLds = (W * 32 * (D * 2 + 32) > W * 16 * (D + 4) * 4 ? W * 32 * (D * 2 + 32) : W * 16 * (D + 4) * 4) + W * 128;

template <typename T, int D, int MOD, int W>
__device__ __forceinline__ void small_block(const Launch& L, uint32_t block, uint8_t* lds) {
  constexpr int kStride = D * 2 + 32;    // bytes of a V row in LDS: 8 rows start in 8 different bank groups
  constexpr int kSteps = D / 32;         // MFMAs of a score
  constexpr int kLoads = D / 16;         // 1 KB loads of 32 V rows
  constexpr int kLanes = D / 8;          // lanes of a row in them
  constexpr int kOut = D / 16;
  constexpr int kMergeStride = D + 4;
  constexpr int kSmallTile = 32 * W;     // positions that the waves take per step
  float(*ml)[16][2] = (float(*)[16][2])(lds + kSmallLds<D, W> - W * 128);
  const AttnParams& a = L.a;
  const uint32_t t = threadIdx.x % (64 * W);
  const uint32_t wave = uniform(t >> 6), lane = t & 63;
  const uint32_t h = block % a.n_kv, item = block / a.n_kv;
  // the division of all sequences' positions, found by every wave alike
  auto tiles_of = [&](uint32_t s, bool* bad, bool* mine) { return small_steps<W>(a, s, bad, mine); };
  Found f;
  bool found;
  if (L.n.planned) {
    found = find_planned(L.ws.plan, a.b.n_seq, item, &f);
  } else {
    uint32_t total = 0, tiles0 = 0;  // (tiles0: of the first 64 sequences, which are not looked at twice)
    bool mine0 = false;
    for (uint32_t s0 = 0; s0 < a.b.n_seq; s0 += 64) {
      const uint32_t s = s0 + lane;
      uint32_t n = 0;
      if (s < a.b.n_seq) {
        bool bad, mine;
        n = tiles_of(s, &bad, &mine);
        if (bad && block == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
        if (s0 == 0) {
          tiles0 = n;
          mine0 = mine;
        }
      }
      total += n;
    }
    total = lane_value(wave_scan(total), 63);
    // (without a launch that joins parts, there are none)
    const uint32_t per_item = L.n.merge ? (total + L.n.item_goal - 1) / L.n.item_goal : total;
    found = find_item(a.b.n_seq, item, [&](uint32_t s) {
      uint32_t n = tiles0;
      bool bad, mine = mine0;
      if (s >= 64) n = tiles_of(s, &bad, &mine);
      return n ? items_of(n, per_item) : mine ? 1u : 0u;
    }, &f);
  }
  if (!found) {
    __syncthreads();  // as often as a neighbour in the same block
    __syncthreads();
    return;
  }
  const uint32_t s = f.s, first = f.first, n_items = f.n;
  bool bad;
  const SeqSpan sq = seq_span(a, s, &bad);
  const uint32_t tiles = sq.end > sq.begin ? (uint32_t)(sq.end - sq.begin + kSmallTile - 1) / kSmallTile : 0;
  const uint32_t part = item - first, share = (tiles + n_items - 1) / n_items;
  const int32_t from = sq.begin + (int32_t)(part * share * kSmallTile);
  const int32_t to = min(sq.end, from + (int32_t)(share * kSmallTile));
  if (!L.n.planned && t == 0 && part == 0 && h == 0) {
    L.ws.plan[2 * s] = first;
    L.ws.plan[2 * s + 1] = n_items;
  }
  // the lane's row
  const uint32_t col = lane & 15, quad = lane >> 4;
  const bool active = col < sq.rows;
  const uint32_t qi = active ? col / a.group : 0, g = active ? col % a.group : 0;
  const uint32_t row = sq.v.q0 + qi, head = h * a.group + g;
  const int32_t pos = sq.p0 + (int32_t)qi;
  const RowSpan span = row_span(pos, sq.v.kv_len, a.window, sq.prefix);
  const RowSpan span0 = row_span(sq.p0, sq.v.kv_len, a.window, sq.prefix);
  const RowSpan span1 = row_span((int32_t)sq.v.kv_len - 1, sq.v.kv_len, a.window, sq.prefix);
  const float slope2 = MOD && a.slopes ? a.slopes[head] * kLog2e : 0.0f;
  vec8<T> q[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; i++) {
    u32x4_t z = {0, 0, 0, 0};
    if (active)
      z = *(const u32x4_t*)((const T*)a.q + (size_t)row * a.q_stride + (size_t)head * D + i * 32 + quad * 8);
    q[i] = __builtin_bit_cast(vec8<T>, z ^ L.sc.flip);
  }
  const float mul = MOD ? 1.0f : L.sc.mul;
  f32x4_t o[kOut];
#pragma unroll
  for (int i = 0; i < kOut; i++) o[i] = f32x4_t{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  uint8_t RLH_LDS* vrows = (uint8_t RLH_LDS*)lds + wave * 32 * kStride;
  u32x4_t kr[2][kSteps], vr[kLoads];
  const uint32_t* table = a.b.table + (size_t)s * a.b.table_stride;
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  // whether the 16 positions at p hold any that a row sees
  auto needed = [&](int32_t p) { return p < to && (p < span1.prefix || p + 16 > span0.lo); };
  auto entry = [&](int32_t p) { return needed(p) ? load_uniform(table, (uint32_t)p >> a.page_shift) : 0u; };
  uint32_t valid = 0;  // of the two groups in the registers
  auto issue = [&](int32_t p, uint32_t e0, uint32_t e1) {
    valid = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int32_t pu = p + 16 * u;
      uint32_t page = u ? e1 : e0;
      bool ok = needed(pu);
      if (ok && page >= a.n_pages) {
        raise(lane == 0 ? a.status : nullptr, RLH_SERVE_BAD_PAGE);
        ok = false;
      }
      if (!ok) page = 0;
      valid |= ok ? 1u << u : 0u;
      const size_t at = ((((size_t)page * a.n_kv + h) << a.page_shift) + (ok ? (uint32_t)pu & page_mask : 0)) * D;
      const T* kp = (const T*)a.pool_k + at;
      const T* vp = (const T*)a.pool_v + at;
#pragma unroll
      for (int i = 0; i < kSteps; i++)
        kr[u][i] = *(const RLH_GLOBAL u32x4_t*)(kp + (col * D + i * 32 + quad * 8));
#pragma unroll
      for (int i = 0; i < kLoads / 2; i++)
        vr[u * (kLoads / 2) + i] = *(const RLH_GLOBAL u32x4_t*)(vp + (i * 512 + lane * 8));
    }
  };
  int32_t p = from + (int32_t)wave * 32;
  if (p < to) {
    issue(p, entry(p), entry(p + 16));
    uint32_t e0 = entry(p + kSmallTile), e1 = entry(p + kSmallTile + 16);
    for (; p < to; p += kSmallTile) {
      const uint32_t ok = valid;
      const bool full = ok == 3 && ((p >= span1.lo && p + 32 <= span0.hi) || p + 32 <= span0.prefix);
      f32x4_t sc[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        sc[u] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kSteps; i++) sc[u] = mfma16(__builtin_bit_cast(vec8<T>, kr[u][i]), q[i], sc[u]);
      }
      uint64_t special = 0;  // V rows with values that a zero would not silence
      if (!full) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
          const uint64_t b = __ballot(any_special<T>(vr[i]));
#pragma unroll
          for (int r = 0; r < 64 / kLanes; r++)
            if (b >> (r * kLanes) & ((1ull << kLanes) - 1)) special |= 1ull << (i * (64 / kLanes) + r);
        }
      }
#pragma unroll
      for (int i = 0; i < kLoads; i++)
        *(RLH_LDS_PTR(u32x4_t)*)(vrows + (i * (64 / kLanes) + lane / kLanes) * kStride + (lane % kLanes) * 16) = vr[i];
      if (p + kSmallTile < to) {
        issue(p + kSmallTile, e0, e1);
        e0 = entry(p + 2 * kSmallTile);
        e1 = entry(p + 2 * kSmallTile + 16);
      }
      __builtin_amdgcn_sched_barrier(0);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int32_t j = p + (i / 4) * 16 + (int32_t)quad * 4 + i % 4;
        x[i] = MOD ? score<MOD>(L.sc, sc[i / 4][i % 4], slope2, (float)(j - pos)) : sc[i / 4][i % 4];
      }
      if (!full) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int32_t j = p + (i / 4) * 16 + (int32_t)quad * 4 + i % 4;
          x[i] = (row_sees(span, j) & (bool)(ok >> (i / 4) & 1)) ? x[i] : -INFINITY;
        }
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
      top = max_across_16(max_across_32(top));
      if constexpr (!MOD) top *= mul;
      if (__ballot(top > m + kSlack)) {
        const float mn = fmaxf(m, top);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int i = 0; i < kOut; i++) o[i] *= f;
        m = mn;
      }
      const float mb = (m == -INFINITY ? 0.0f : m) - kLift<T>;
      vec8<T> pr;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], mul, -mb));
        l += x[i];
        pr[i] = (T)x[i];
      }
      while (special) {
        // such a row is added to the rows that see it, one by one, and
        // silenced for the product
        const int32_t r = (int32_t)__builtin_ctzll(special);
        special &= special - 1;
        const int32_t j = p + r;
        const bool see = (ok >> (r / 16) & 1) && row_sees(span, j);
        const float pv = element<T>(pr, (uint32_t)(r / 16 * 4 + r % 4), (int)(col + 16 * (uint32_t)(r % 16 / 4)));
#pragma unroll
        for (int i = 0; i < kOut; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float v = (float)*(RLH_LDS_PTR(T)*)(vrows + r * kStride + (i * 16 + quad * 4 + e) * 2);
            if (see) o[i][e] = fmaf(pv, v, o[i][e]);
          }
        if (lane < (uint32_t)kLanes) *(RLH_LDS_PTR(u32x4_t)*)(vrows + r * kStride + lane * 16) = u32x4_t{0, 0, 0, 0};
      }
      const uint8_t RLH_LDS* vc = vrows + (quad * 4 + col / 4) * kStride + col % 4 * 8;
#pragma unroll
      for (int i = 0; i < kOut; i++) o[i] = mfma16(read_columns<T>(vc + i * 32, vc + 16 * kStride + i * 32), pr, o[i]);
    }
  }
  l = sum_across_16(sum_across_32(l));
  // the waves' results
  __syncthreads();
  float* ol = (float*)lds;
#pragma unroll
  for (int i = 0; i < kOut; i++) *(f32x4_t*)(ol + (wave * 16 + col) * kMergeStride + i * 16 + quad * 4) = o[i];
  if (quad == 0) {
    ml[wave][col][0] = m;
    ml[wave][col][1] = l;
  }
  __syncthreads();
  constexpr int kRowLanes = 4 * W, N = D / kRowLanes;  // threads and values of a row
  const uint32_t r = t / kRowLanes, c0 = (t % kRowLanes) * N;
  if (r >= sq.rows) return;
  float mm = -INFINITY, ls = 0.0f, acc[N] = {};
#pragma unroll
  for (int w = 0; w < W; w++) mm = fmaxf(mm, ml[w][r][0]);
  const float mb = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
  for (int w = 0; w < W; w++) {
    const float f = __builtin_amdgcn_exp2f(ml[w][r][0] - mb);
    ls += ml[w][r][1] * f;
#pragma unroll
    for (int i = 0; i < N; i++) acc[i] = fmaf(ol[(w * 16 + r) * kMergeStride + c0 + i], f, acc[i]);
  }
  if (n_items == 1 && a.shared_len == 0) {
    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
    T* dst = (T*)a.out + (size_t)(sq.v.q0 + r / a.group) * a.out_stride + (size_t)(h * a.group + r % a.group) * D + c0;
    typedef T VO __attribute__((ext_vector_type(N)));
    VO v;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (T)(acc[i] * inv);
    *(VO*)dst = v;
  } else {
    const size_t at = ((size_t)item * a.n_kv + h) * kSmallRows + r;
    float* dst = L.ws.item_o + at * D + c0;
#pragma unroll
    for (int i = 0; i < N; i++) dst[i] = acc[i];
    if (c0 == 0) {
      L.ws.item_ml[2 * at] = mm;
      L.ws.item_ml[2 * at + 1] = ls;
    }
  }
}

template <typename T, int D, int MOD, int W>
__global__ void __launch_bounds__(64 * W, 2) k_attn_small(Launch L) {
  extern __shared__ __align__(1024) uint8_t lds[];
  small_block<T, D, MOD, W>(L, blockIdx.x, lds);
}

// ---- many rows: prompts, and the shared prefix of the whole batch ------------------
// A block takes 256 rows of one KV head (rows are tokens times heads per KV
// head, so heads that share K and V share a tile) and walks 64 positions at
// a time; K and V are copied into LDS by DMA, one step ahead, in 16-byte
// pieces that are exchanged within a row so that the products' reads meet no
// bank twice. Each of eight waves has 32 rows: scores are K times Q^T
// (32x32x16: positions down, rows across), so that a row is a lane column as
// above. What bounds it: a step's 32 MFMAs take a wave 1024 cycles of its SIMD
// and its exponentials, maxima and sums as many; within a wave they are one
// chain, and the two waves of a SIMD overlap little of it (a step takes 2.3 us,
// the sum of both waves' 4096 cycles 1.7). Copies are issued at 48 cycles a
// KB, so four waves per tile would spend 1550 cycles a step on them. 4096
// tokens of 64 heads: 275 GFLOP in 300 us, 916 TFLOP/s (a product of 16384^3
// reaches 1357). In a row of passes it is 340 us; there, tiles of 128 rows took
// 382, operand reads that do not run ahead of the products 349. A cap adds an exponential and a reciprocal per
// score; a bias is linear in the position, so that a row's share at the step's
// first position is kept out of the scores and joins the running maximum only
// (5 prompts of 6895 tokens with a bias: 147 us with it in each score, 104).
template <int D>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  return D == 128 ? ((r & 3) << 2 | (r >> 2 & 3)) : ((r >> 1 & 1) << 2 | (r >> 2 & 3));
}

// Tiles of sequence s.
__device__ __forceinline__ uint32_t tiles_of_seq(const Launch& L, uint32_t s) {
  bool bad;
  const SeqView v = load_seq(L.a.b, s, &bad);
  const uint32_t r = v.ok ? v.q_len * L.a.group : 0;
  return r > L.n.small_rows ? (r + kTileRows - 1) / kTileRows : 0u;
}

struct TileShared {
  uint64_t special[2];  // positions of a step whose V row holds infinities or NaN
  int32_t ranges[kTileWaves][8];
};
template <int D>
constexpr uint32_t kTileLds = 4 * kTileKv * D * 2 + sizeof(TileShared);

template <typename T, int D, int MOD>
__device__ __forceinline__ void tile_block(const Launch& L, uint32_t block, bool prefix, uint8_t* lds) {
  constexpr int kRowB = D * 2;
  constexpr int kBuf = kTileKv * kRowB;   // bytes of a K or V step
  constexpr int kSteps = D / 16;
  constexpr int kOut = D / 32;
  constexpr int kLanes = D / 8;           // lanes of a row in a copy
  constexpr int kThreads = 64 * kTileWaves;
  constexpr int kMine = kTileKv / kTileWaves;           // positions of a step that a wave copies
  constexpr int kCopies = kMine / (64 / kLanes);        // in 1 KB pieces
  // K, V of two steps first
  TileShared& sh = *(TileShared*)(lds + 4 * kBuf);
  uint64_t* special = sh.special;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(RLH_LDS uint8_t*)lds;
  const AttnParams& a = L.a;
  const uint32_t t = threadIdx.x;
  const uint32_t wave = uniform(t >> 6), lane = t & 63;
  const uint32_t h = block % a.n_kv, of_head = block / a.n_kv;
  uint32_t parts = prefix ? L.n.prefix_parts : L.n.tile_parts, tile = of_head / parts, part = of_head % parts;
  if (prefix && tile >= L.n.prefix_tiles - 1) {
    tile = L.n.prefix_tiles - 1;
    part = of_head - tile * parts;
    parts = L.n.last_parts;
  }
  // the tile's sequence (own positions), or all rows (the prefix)
  uint32_t s = 0, row0 = 0, rows = 0;
  if (prefix) {
    row0 = tile * kTileRows;
    rows = a.b.n_rows * a.group;
  } else {
    if (block == 0 && !L.n.planned)
      for (uint32_t i = t; i < a.b.n_seq; i += kThreads) {
        bool bad;
        load_seq(a.b, i, &bad);
        if (bad) raise(a.status, RLH_SERVE_BAD_SEQ);
      }
    Found f;
    if (L.n.planned ? !find_planned(L.ws.tiles, a.b.n_seq, tile, &f)
                    : !find_item(a.b.n_seq, tile, [&](uint32_t i) { return tiles_of_seq(L, i); }, &f))
      return;
    s = f.s;
    row0 = (f.n - 1 - (tile - f.first)) * kTileRows;  // the last rows, with the most positions, first
    bool bad;
    rows = load_seq(a.b, s, &bad).q_len * a.group;
  }
  // the lane's row
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t rr = row0 + wave * 32 + col;
  bool active = rr < rows;
  uint32_t row = rr / a.group, g = rr % a.group, sq = s;
  if (prefix) {
    uint32_t lo = 0, hi = a.b.n_seq;  // as many sequences end at or before the row as come before its own
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (active && a.b.q_start[mid + 1] <= row)
        lo = mid + 1;
      else
        hi = mid;
    }
    sq = lo;
    active = active && sq < a.b.n_seq;
  }
  SeqView sv{};
  if (active) {
    bool bad;
    sv = load_seq(a.b, sq, &bad);
    if (!prefix) row += sv.q0;
    active = sv.ok && row >= sv.q0 && row < sv.q0 + sv.q_len;
  }
  const int32_t pos = (int32_t)(sv.kv_len - sv.q_len) + (int32_t)(row - sv.q0);
  const uint32_t head = h * a.group + g;
  const int32_t limit = prefix ? min((int32_t)a.shared_len, (int32_t)sv.kv_len) : (int32_t)sv.kv_len;
  RowSpan span{0, 0, 0};
  if (active) {
    span = row_span(pos, sv.kv_len, a.window, a.prefix_len ? a.prefix_len[sq] : 0);
    span.hi = min(span.hi, limit);
    span.prefix = min(span.prefix, limit);
  }
  // positions that the wave's rows all see lie in [w_lo, w_hi) or below
  // w_prefix; those that any sees in [b_lo, b_hi)
  int32_t w_lo = active ? span.lo : 0, w_hi = active ? span.hi : 0x7fffffff, w_prefix = active ? span.prefix : 0x7fffffff;
  int32_t b_lo = active ? max(span_begin(span), prefix ? 0 : (int32_t)a.shared_len) : 0x7fffffff;
  int32_t b_hi = active ? span_end(span) : 0;
  int32_t any_prefix = active ? span.prefix : 0, min_lo = active ? span.lo : 0x7fffffff;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    w_lo = max(w_lo, __shfl_xor(w_lo, d));
    w_hi = min(w_hi, __shfl_xor(w_hi, d));
    w_prefix = min(w_prefix, __shfl_xor(w_prefix, d));
    b_lo = min(b_lo, __shfl_xor(b_lo, d));
    b_hi = max(b_hi, __shfl_xor(b_hi, d));
    any_prefix = max(any_prefix, __shfl_xor(any_prefix, d));
    min_lo = min(min_lo, __shfl_xor(min_lo, d));
  }
  w_lo = (int32_t)uniform(w_lo);
  w_hi = (int32_t)uniform(w_hi);
  w_prefix = (int32_t)uniform(w_prefix);
  const int32_t v_lo = (int32_t)uniform(b_lo), v_hi = (int32_t)uniform(b_hi);  // the wave's
  if (lane == 0) {
    int32_t* r = sh.ranges[wave];
    r[0] = v_lo;
    r[1] = v_hi;
    r[2] = any_prefix;
    r[3] = min_lo;
    r[4] = w_lo;
    r[5] = w_hi;
    r[6] = w_prefix;
  }
  __syncthreads();
  int32_t t_lo = 0x7fffffff, t_hi = 0, t_prefix = 0, t_min_lo = 0x7fffffff;  // the block's
  int32_t c_lo = 0, c_hi = 0x7fffffff, c_prefix = 0x7fffffff;
#pragma unroll
  for (int w = 0; w < kTileWaves; w++) {
    const int32_t* r = sh.ranges[w];
    t_lo = min(t_lo, r[0]);
    t_hi = max(t_hi, r[1]);
    t_prefix = max(t_prefix, r[2]);
    t_min_lo = min(t_min_lo, r[3]);
    c_lo = max(c_lo, r[4]);
    c_hi = min(c_hi, r[5]);
    c_prefix = min(c_prefix, r[6]);
  }
  c_lo = (int32_t)uniform(c_lo);
  c_hi = (int32_t)uniform(c_hi);
  c_prefix = (int32_t)uniform(c_prefix);
  t_lo = (int32_t)uniform(t_lo & ~15);
  t_hi = (int32_t)uniform(t_hi);
  t_prefix = (int32_t)uniform(t_prefix);
  t_min_lo = (int32_t)uniform(t_min_lo);
  const uint32_t n_steps = t_hi > t_lo ? (uint32_t)(t_hi - t_lo + kTileKv - 1) / kTileKv : 0;
  const uint32_t st0 = (uint32_t)((uint64_t)n_steps * part / parts), st1 = (uint32_t)((uint64_t)n_steps * (part + 1) / parts);

  const float slope2 = MOD && a.slopes && active ? a.slopes[head] * kLog2e : 0.0f;
  vec8<T> q[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; i++) {
    u32x4_t z = {0, 0, 0, 0};
    if (active) z = *(const u32x4_t*)((const T*)a.q + (size_t)row * a.q_stride + (size_t)head * D + i * 16 + half * 8);
    q[i] = __builtin_bit_cast(vec8<T>, z ^ L.sc.flip);
  }
  const float mul = MOD ? 1.0f : L.sc.mul;
  f32x16_t o[kOut];
#pragma unroll
  for (int i = 0; i < kOut; i++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[i][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  const uint32_t* table = prefix ? a.shared_table : a.b.table + (size_t)s * a.b.table_stride;
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  // Page ids of 16 steps, a group of 16 positions per lane (the id, or none),
  // loaded some steps before their first use
  constexpr uint32_t kNone = 0xffffffffu;
  auto look_up = [&](uint32_t step) -> uint32_t {
    const int32_t g = t_lo + (int32_t)step * kTileKv + 16 * (int32_t)lane;
    // whether the group holds positions that a row sees
    if (!((g < t_hi) & ((g < t_prefix) | (g + 16 > t_min_lo)))) return kNone;
    const uint32_t e = table[(uint32_t)g >> a.page_shift];
    if (e < a.n_pages) return e;
    if (wave == 0) raise(a.status, RLH_SERVE_BAD_PAGE);
    return kNone;
  };
  uint32_t from[kCopies];  // of the wave's positions, what each lane copies
#pragma unroll
  for (int i = 0; i < kCopies; i++) {
    const uint32_t r = wave * kMine + i * (64 / kLanes) + lane / kLanes;  // of the step
    from[i] = r % 16 * D + ((lane % kLanes) ^ swizzle<D>(r)) * 8;
  }
  // copies the wave's positions of the step at p, whose groups are lanes
  // 4 k .. 4 k + 3 of `pages`
  auto copy = [&](int32_t p, uint32_t pages, uint32_t k, uint32_t buf) {
    const uint32_t u = wave * kMine / 16;
    const uint32_t page = lane_value(pages, (int)(4 * k + u));
    const bool exists = page != kNone;
    const uint32_t slot = exists ? (uint32_t)(p + 16 * (int32_t)u) & page_mask : 0u;
    const size_t at = ((((size_t)(exists ? page : 0u) * a.n_kv + h) << a.page_shift) + slot) * D;
    const uint32_t dst = lds0 + buf * 2 * kBuf + wave * kMine * kRowB;
#pragma unroll
    for (int i = 0; i < kCopies; i++) {
      copy_to_lds((const T*)a.pool_k + at + from[i], dst + i * 1024);
      copy_to_lds((const T*)a.pool_v + at + from[i], dst + i * 1024 + kBuf);
    }
  };
  // Two waves share a SIMD; left alone they go through products and
  // exponentials in step and take turns at both.
  if (wave >= kTileWaves / 2) __builtin_amdgcn_s_setprio(2);
  // operands: K's row 32 u + col, values 16 i + 8 half + 0..7; V's rows 16 ks +
  // 4 half + 0..3 and + 8, by columns 32 i + 16 (lane / 16 % 2) + 0..15
  const uint32_t va = half * 4 + lane % 16 / 4, vb8 = va + 8;
  uint32_t v_at[2][kOut], k_at[kSteps];
#pragma unroll
  for (int i = 0; i < kOut; i++) {
    const uint32_t d = i * 32 + (lane >> 4 & 1) * 16 + lane % 4 * 4;
    v_at[0][i] = va * kRowB + ((d / 8) ^ swizzle<D>(va)) * 16 + d % 8 * 2;
    v_at[1][i] = vb8 * kRowB + ((d / 8) ^ swizzle<D>(vb8)) * 16 + d % 8 * 2;
  }
#pragma unroll
  for (int i = 0; i < kSteps; i++) k_at[i] = col * kRowB + ((2 * i + half) ^ swizzle<D>(col)) * 16;
  auto load_v = [&](const uint8_t RLH_LDS* vb, int ks, vec8<T> (&f)[kOut]) {
#pragma unroll
    for (int i = 0; i < kOut; i++)
      f[i] = read_columns<T>(vb + v_at[0][i] + ks * 16 * kRowB, vb + v_at[1][i] + ks * 16 * kRowB);
  };
  auto load_k = [&](const uint8_t RLH_LDS* kb, int u, vec8<T> (&f)[kSteps]) {
#pragma unroll
    for (int i = 0; i < kSteps; i++)
      f[i] = __builtin_bit_cast(vec8<T>, *(const RLH_LDS_PTR(u32x4_t)*)(kb + k_at[i] + u * 32 * kRowB));
  };
  uint32_t pages = kNone, next_pages = kNone;
  uint64_t exist = 0;  // the groups of `pages` whose page exists
  if (st0 < st1) {
    pages = look_up(st0);
    exist = __ballot(pages != kNone);
    copy(t_lo + (int32_t)st0 * kTileKv, pages, 0, 0);
  }
  for (uint32_t st = st0; st < st1; st++) {
    const uint32_t buf = (st - st0) & 1;
    const int32_t p = t_lo + (int32_t)st * kTileKv;
    const uint32_t k = (st - st0) & 15;
    const uint32_t ok = (uint32_t)(exist >> (4 * k)) & 15;
    if (t == 0) special[buf] = 0;  // last read two barriers ago
    wait_vmcnt<0>();               // this wave's copies of the step have landed
    lds_barrier();                 // ... everyone's; every wave is done with the other buffer
    if (k == 8) next_pages = look_up(st + 8);
    if (k == 15) {
      pages = next_pages;
      exist = __ballot(pages != kNone);
    }
    if (st + 1 < st1) copy(p + kTileKv, pages, (k + 1) & 15, buf ^ 1);
    const uint8_t RLH_LDS* kb = (const uint8_t RLH_LDS*)lds + buf * 2 * kBuf;
    uint8_t RLH_LDS* vb = (uint8_t RLH_LDS*)lds + buf * 2 * kBuf + kBuf;
    const bool full = ok == 15 && ((p >= w_lo && p + kTileKv <= w_hi) || p + kTileKv <= w_prefix);
    const bool none = p >= v_hi || p + kTileKv <= v_lo;
    // values that a zero would not silence, in steps that not every row of
    // the block sees whole
    uint64_t odd = 0;
    if (!(ok == 15 && ((p >= c_lo && p + kTileKv <= c_hi) || p + kTileKv <= c_prefix))) {
#pragma unroll
      for (int i = 0; i < kBuf / (kThreads * 16); i++) {
        const uint32_t at = (i * kThreads + t) * 16;
        if (any_special<T>(*(const RLH_LDS_PTR(u32x4_t)*)(vb + at)))
          atomicOr((unsigned long long*)&special[buf], 1ull << (at / kRowB));
      }
      lds_barrier();
      odd = special[buf];
    }
    f32x16_t sc[2];
    vec8<T> pr[4];
    if (!none) {
      // reads well ahead of the products (one read takes some 250 cycles)
      vec8<T> k0[kSteps], k1[kSteps];
      load_k(kb, 0, k0);
      load_k(kb, 1, k1);
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) sc[u][e] = 0.0f;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kSteps; i++) sc[0] = mfma32(k0[i], q[i], sc[0]);
#pragma unroll
      for (int i = 0; i < kSteps; i++) sc[1] = mfma32(k1[i], q[i], sc[1]);
      // the lane's first position; the others are constants away (opaque, so
      // that 32 of them are not kept in registers from step to step)
      int32_t j0 = p + (int32_t)half * 4;
      asm volatile("" : "+v"(j0));
      float far = 0.0f;  // what all of the row's scores lack
      if constexpr (MOD) {
        if constexpr (MOD == kWideCap) {
#pragma unroll
          for (int i = 0; i < 32; i++) sc[i / 16][i % 16] = capped_wide(L.sc, sc[i / 16][i % 16]);
        } else if (L.sc.capped) {
#pragma unroll
          for (int i = 0; i < 32; i++) sc[i / 16][i % 16] = capped(L.sc, sc[i / 16][i % 16]);
        }
        if (L.sc.biased) {
          // slope * distance = far + near + slope * (0 .. 59): far that of the
          // step's first position, near the rest up to the lane's first
          far = slope2 * (float)(p - pos);
          const float near = fmaf(slope2, (float)(j0 - pos), -far);
          const float mul1 = L.sc.capped ? 1.0f : L.sc.mul;
#pragma unroll
          for (int i = 0; i < 32; i++)
            sc[i / 16][i % 16] = fmaf(sc[i / 16][i % 16], mul1, fmaf(slope2, (float)(i / 4 * 8 + i % 4), near));
        }
      }
      if (!full) {
        const int32_t lo = span.lo - j0, hi = span.hi - j0, pre = span.prefix - j0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
          const int32_t d = i / 4 * 8 + i % 4;
          const bool see = ((d >= lo) & (d < hi)) | (d < pre);
          sc[i / 16][i % 16] = (see & (bool)(ok >> (i / 8) & 1)) ? sc[i / 16][i % 16] : -INFINITY;
        }
      }
      float top = sc[0][0];
#pragma unroll
      for (int i = 1; i < 32; i++) top = fmaxf(top, sc[i / 16][i % 16]);
      top = max_across_32(top);
      top = MOD ? top + far : top * mul;
      if (__ballot(top > m + kSlack)) {
        const float mn = fmaxf(m, top);
        const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int i = 0; i < kOut; i++) o[i] *= f;
        m = mn;
      }
      const float mb = (m == -INFINITY ? 0.0f : m) - far - kLift<T>;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float x = __builtin_amdgcn_exp2f(fmaf(sc[u][e], mul, -mb));
          l += x;
          pr[2 * u + e / 8][e % 8] = (T)x;
        }
    }
    if (odd) {
      if (!none) {
        for (uint64_t left = odd; left; left &= left - 1) {
          const int32_t r = (int32_t)__builtin_ctzll(left), j = p + r;
          const bool see = active && (ok >> (r / 16) & 1) && row_sees(span, j);
          float pv = 0.0f;
#pragma unroll
          for (int ks = 0; ks < 4; ks++) {
            const float c = element<T>(pr[ks], (uint32_t)(r % 16 / 8 * 4 + r % 4), (int)(col + 32 * (uint32_t)(r % 8 / 4)));
            if (ks == r / 16) pv = c;
          }
#pragma unroll
          for (int i = 0; i < kOut; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const uint32_t d = i * 32 + (e / 4) * 8 + half * 4 + e % 4;
              const float v = (float)*(const RLH_LDS_PTR(T)*)(vb + r * kRowB + ((d / 8) ^ swizzle<D>(r)) * 16 + d % 8 * 2);
              if (see) o[i][e] = fmaf(pv, v, o[i][e]);
            }
        }
      }
      lds_barrier();
      for (uint64_t left = odd; left; left &= left - 1) {
        const uint32_t r = (uint32_t)__builtin_ctzll(left);
        if (t < (uint32_t)kLanes) *(RLH_LDS_PTR(u32x4_t)*)(vb + r * kRowB + t * 16) = u32x4_t{0, 0, 0, 0};
      }
      lds_barrier();
    }
    if (!none) {
      vec8<T> f[2][kOut];
      load_v(vb, 0, f[0]);
      load_v(vb, 1, f[1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < 4; ks++) {
#pragma unroll
        for (int i = 0; i < kOut; i++) o[i] = mfma32(f[ks % 2][i], pr[ks], o[i]);
        if (ks < 2) load_v(vb, ks + 2, f[ks % 2]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  l = sum_across_32(l);
  if (!active) return;
  if (!prefix && parts == 1 && a.shared_len == 0) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* dst = (T*)a.out + (size_t)row * a.out_stride + (size_t)head * D;
#pragma unroll
    for (int i = 0; i < kOut; i++)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        vec4<T> v;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = (T)(o[i][e + k] * inv);
        *(vec4<T>*)(dst + i * 32 + (e / 4) * 8 + half * 4) = v;
      }
  } else {
    const size_t at = ((size_t)part * a.b.n_rows + row) * a.n_head + head;
    float* dst = (prefix ? L.ws.prefix_o : L.ws.tile_o) + at * D;
    float* mlp = (prefix ? L.ws.prefix_ml : L.ws.tile_ml) + at * 2;
#pragma unroll
    for (int i = 0; i < kOut; i++)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4_t*)(dst + i * 32 + (e / 4) * 8 + half * 4) = f32x4_t{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
    if (half == 0) {
      mlp[0] = m;
      mlp[1] = l;
    }
  }
}

// Prefix tiles, tiles and items of few rows in one launch, long blocks first:
// each kind leaves parts of the card idle that the others fill (64 tokens of
// 32 heads behind 4096 shared positions: 28 us, in launches of their own
// 20 + 17; 72 of 64 heads behind 16384: 70 us, apart 65 + 14 + 5; a prompt
// alone loses 1 % by it).
template <typename T, int D, int MOD>
__global__ void __launch_bounds__(64 * kTileWaves, 2) k_attn_mixed(Launch L) {
  extern __shared__ __align__(1024) uint8_t lds[];
  const uint32_t n_prefix = prefix_blocks(L.n) * L.a.n_kv;
  const uint32_t n_tiles = n_prefix + L.n.tiles * L.n.tile_parts * L.a.n_kv;
  const uint32_t b = blockIdx.x;
  if (b < n_tiles) {
    tile_block<T, D, MOD>(L, b < n_prefix ? b : b - n_prefix, b < n_prefix, lds);
  } else {  // two items, of four waves each
    const uint32_t half = uniform(threadIdx.x / kThreads);
    small_block<T, D, MOD, kWaves>(L, 2 * (b - n_tiles) + half, lds + half * kSmallLds<D, kWaves>);
  }
}

// ---- joining the parts of a row ------------------------------------------------------
// A wave takes a row of a query head, its four groups of 16 lanes every
// fourth part: all maxima at once, then the parts' values, four parts' loads
// of a group at a time. Bound by latency (a part of a row is 512 bytes at a
// place of its own): 4 us for a single sequence, 8 for 2048 rows and heads of
// 17 parts (36 MB).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) k_attn_merge(Launch L) {
  constexpr int N = D / 16;   // values per lane
  constexpr uint32_t kAhead = 4;
  const AttnParams& a = L.a;
  const uint32_t lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  uint32_t s = 0, row, head, r;
  SeqView sv;
  bool bad;
  if (L.n.merge_small) {  // blocks: (sequence, four rows, KV head)
    const uint32_t h = blockIdx.x % a.n_kv, i = blockIdx.x / a.n_kv;
    s = i / L.n.merge_rows;
    sv = load_seq(a.b, s, &bad);
    r = i % L.n.merge_rows * kWaves + wave;
    row = sv.q0 + r / a.group;
    head = h * a.group + r % a.group;
  } else {  // waves: (row, head)
    const uint32_t w = blockIdx.x * kWaves + wave;
    row = w / a.n_head;
    head = w % a.n_head;
    if (row >= a.b.n_rows) return;
    s = count_upto(a.b.q_start + 1, 1, a.b.n_seq, row);
    if (s >= a.b.n_seq) return;
    sv = load_seq(a.b, s, &bad);
    if (row < sv.q0) return;
    r = (row - sv.q0) * a.group + head % a.group;
  }
  if (!sv.ok || r >= sv.q_len * a.group) return;
  const bool small = sv.q_len * a.group <= L.n.small_rows;
  if (L.n.merge_small && !small) return;
  const uint32_t in_head = row * a.group + head % a.group;  // among all rows of its KV head
  const uint32_t n_prefix = !a.shared_len                                       ? 0
                            : in_head / kTileRows + 1 < L.n.prefix_tiles ? L.n.prefix_parts
                                                                        : L.n.last_parts;
  const uint32_t first = small ? load_uniform(L.ws.plan, 2 * s) : 0;
  const uint32_t n_own = small ? load_uniform(L.ws.plan, 2 * s + 1) : L.n.tile_parts;
  if (n_prefix == 0 && n_own == 1) return;  // written already
  const uint32_t h = head / a.group;
  const size_t rh = (size_t)row * a.n_head + head, all = (size_t)a.b.n_rows * a.n_head;
  const uint32_t n = n_prefix + n_own;
  auto place = [&](uint32_t i, const float** o, const float** ml) {
    size_t at;
    if (i < n_prefix) {
      at = i * all + rh;
      *o = L.ws.prefix_o;
      *ml = L.ws.prefix_ml;
    } else if (small) {
      at = ((size_t)(first + i - n_prefix) * a.n_kv + h) * kSmallRows + r;
      *o = L.ws.item_o;
      *ml = L.ws.item_ml;
    } else {
      at = (i - n_prefix) * all + rh;
      *o = L.ws.tile_o;
      *ml = L.ws.tile_ml;
    }
    *o += at * D;
    *ml += at * 2;
  };
  float m = -INFINITY;
  for (uint32_t i = lane; i < n; i += 64) {
    const float *o, *ml;
    place(i, &o, &ml);
    m = fmaxf(m, ml[0]);
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  m = max_across_16(max_across_32(m));
  const float mb = m == -INFINITY ? 0.0f : m;
  const uint32_t quad = lane / 16, c0 = lane % 16 * N;
  float l = 0.0f, acc[N] = {};
  for (uint32_t i0 = quad; i0 < n; i0 += 4 * kAhead) {
    f32x4_t v[kAhead][N / 4];
    float mi[kAhead], li[kAhead];
#pragma unroll
    for (uint32_t q = 0; q < kAhead; q++) {
      const uint32_t i = i0 + 4 * q;
      const float *o, *ml;
      place(i < n ? i : i0, &o, &ml);
      mi[q] = i < n ? ml[0] : -INFINITY;
      li[q] = ml[1];
#pragma unroll
      for (int k = 0; k < N / 4; k++) v[q][k] = *(const f32x4_t*)(o + c0 + 4 * k);
    }
#pragma unroll
    for (uint32_t q = 0; q < kAhead; q++) {
      if (i0 + 4 * q >= n) continue;
      const float f = __builtin_amdgcn_exp2f(mi[q] - mb);
      l = fmaf(li[q], f, l);
#pragma unroll
      for (int k = 0; k < N; k++) acc[k] = fmaf(v[q][k / 4][k % 4], f, acc[k]);
    }
  }
  l = sum_across_16(sum_across_32(l));
#pragma unroll
  for (int k = 0; k < N; k++) acc[k] = sum_across_16(sum_across_32(acc[k]));
  if (quad != 0) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  typedef T VO __attribute__((ext_vector_type(N)));
  VO v;
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = (T)(acc[i] * inv);
  *(VO*)((T*)a.out + (size_t)row * a.out_stride + (size_t)head * D + c0) = v;
}

// Up to so many positions, and while all blocks run at once, a sequence of few
// rows is not divided: its block then has eight waves (a step of 256 positions
// takes 2 us) and there is no second launch (8 sequences of 250: 8.6 us
// instead of 7.0 + 4.0, of 500: 10.6 instead of 6.9 + 4.0, of 777: 12.6
// instead of 7.7 + 4.2; 61 of 500, in 488 blocks: 26.4 instead of 24.4 + 4.8,
// 128 of 250: 37.3 instead of 27.6 + 3.8).
constexpr uint32_t kWhole = 512;
// ---- many sequences -------------------------------------------------------------------
// Where each sequence's items and tiles begin, by one block. Up to kPlanned
// sequences every wave of the other kernels finds that out by itself, which
// costs less than a launch; beyond, their loops over all sequences would take
// longer than the attention (2048 tokens of 32 heads over 8 of 128, 300
// positions each: 5 + 448 us instead of 1024).
constexpr uint32_t kPlanned = 256;
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(kPlanThreads) k_attn_plan(Launch L) {
  __shared__ uint32_t sums[2][kPlanThreads / 64];
  const AttnParams& a = L.a;
  const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63;
  // the inclusive sums over the block of two values per thread, and the whole
  auto scan = [&](uint32_t (&x)[2], uint32_t (&all)[2]) {
#pragma unroll
    for (int i = 0; i < 2; i++) x[i] = wave_scan(x[i]);
    __syncthreads();
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < 2; i++) sums[i][wave] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
      all[i] = 0;
      for (uint32_t w = 0; w < kPlanThreads / 64; w++) {
        const uint32_t v = sums[i][w];
        x[i] += w < wave ? v : 0u;
        all[i] += v;
      }
    }
  };
  uint32_t per_item = 0;
  if (L.n.small) {
    uint32_t mine_all = 0;  // of up to 64 sequences
    for (uint32_t s = t; s < a.b.n_seq; s += kPlanThreads) {
      bool bad, mine;
      mine_all += small_steps<kWaves>(a, s, &bad, &mine);
    }
    uint32_t n[2] = {mine_all & 0xffff, mine_all >> 16}, all[2];
    scan(n, all);
    const uint64_t total = all[0] + ((uint64_t)all[1] << 16);
    per_item = steps_per_item(total, L.n.merge ? L.n.item_goal : 1);
  }
  uint32_t before[2] = {0, 0};
  for (uint32_t s0 = 0; s0 < a.b.n_seq; s0 += kPlanThreads) {
    const uint32_t s = s0 + t;
    uint32_t n[2] = {0, 0}, all[2];
    if (s < a.b.n_seq) {
      bool bad, mine;
      const uint32_t steps = small_steps<kWaves>(a, s, &bad, &mine);
      if (bad) raise(a.status, RLH_SERVE_BAD_SEQ);
      if (L.n.small) n[0] = steps ? items_of(steps, per_item) : mine ? 1u : 0u;
      if (L.n.tiled) n[1] = tiles_of_seq(L, s);
    }
    uint32_t upto[2] = {n[0], n[1]};
    scan(upto, all);
    if (s < a.b.n_seq)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t* p = i ? L.ws.tiles : L.ws.plan;
        if (i ? L.n.tiled : L.n.small) {
          p[2 * s] = before[i] + upto[i] - n[i];
          p[2 * s + 1] = n[i];
        }
      }
#pragma unroll
    for (int i = 0; i < 2; i++) before[i] += all[i];
  }
}

// Blocks that the small kernel's work is divided into: three to a CU. So many
// run at once with cap or bias (162 registers) and for head_dim 64, two
// without at 128 (173).
constexpr uint32_t kSmallBlocks = 768;

uint32_t item_goal(uint32_t n_head_kv) { return std::max(1u, kSmallBlocks / n_head_kv); }

// Parts that the positions of `blocks` tiles are divided into: as many as let
// all blocks run at once (one to a CU), of at least 256 positions (of 128,
// what 64 tokens behind 4096 shared positions take grows from 33 + 8 us to
// 41 + 11).
uint32_t tile_parts(uint64_t blocks, uint64_t positions) {
  if (blocks == 0) return 1;
  return (uint32_t)std::max<uint64_t>(1, std::min(256 / blocks, positions / 256));
}

// A score in units of log 2 per unit of the dot product (of 2 / softcap with a cap).
float score_factor(const rlh_attn_args& args) {
  const float scale = fabsf(args.scale);
  return args.softcap > 0.0f ? 2.0f * scale / fminf(args.softcap, kMostCap) * kLog2e : scale * kLog2e;
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
  if (overlaps_pool(*kv, args->out, row_bytes_span(seqs->n_rows, args->out_stride, w, 2)))
    return serve_error(RLH_EINVAL, "out overlaps the pool");
  if (!isfinite(score_factor(*args))) return serve_error(RLH_EINVAL, "scale, or scale / softcap, is out of range");
  return RLH_OK;
}

// How the work of a call is divided, from sizes that the host knows.
Sizes attn_sizes(const rlh_kv_pages& kv, const rlh_seqs& q, const rlh_attn_args& args) {
  Sizes n{};
  const uint64_t group = args.n_head / kv.n_head_kv, rows = (uint64_t)q.n_rows * group;
  const uint64_t own = q.max_kv > args.shared_len ? q.max_kv - args.shared_len : 0;
  n.tiled = q.max_q * group > kSmallRows;
  // a single sequence goes to one of the two kernels as a whole
  n.small = group <= kSmallRows && !(n.tiled && q.n_seq == 1);
  n.small_rows = n.small ? kSmallRows : 0;
  if (n.small) {
    n.whole = !n.tiled && !args.shared_len && q.max_kv <= kWhole && q.n_seq * kv.n_head_kv <= 256;
    n.item_goal = n.whole ? 1 : item_goal(kv.n_head_kv);
    n.items = q.n_seq + (n.whole ? 0 : n.item_goal);
  }
  if (n.tiled) {
    n.tiles = (uint32_t)(rows / kTileRows + std::min<uint64_t>(q.n_seq, rows / (n.small_rows + 1)));
    n.tile_parts = tile_parts((uint64_t)n.tiles * kv.n_head_kv, own);
  }
  if (args.shared_len) {
    n.prefix_tiles = (uint32_t)((rows + kTileRows - 1) / kTileRows);
    n.prefix_parts = n.last_parts = tile_parts((uint64_t)n.prefix_tiles * kv.n_head_kv, args.shared_len);
    // A last tile of up to 128 rows has one wave per SIMD, whose steps take
    // about 0.55 of the time, and is divided into fewer parts (576 rows of a
    // KV head against 16384 positions, the only size it was measured at: 12, 12
    // and 8 parts instead of 10 each, 70 us instead of 75).
    const uint64_t most = 256 / kv.n_head_kv, last = rows - (uint64_t)(n.prefix_tiles - 1) * kTileRows;
    const uint64_t p = std::min<uint64_t>(most * 20 / (20 * n.prefix_tiles - 9), args.shared_len / 256);
    if (n.prefix_tiles > 1 && last <= kTileRows / 2 && p > n.prefix_parts) {
      n.prefix_parts = (uint32_t)p;
      n.last_parts = (uint32_t)std::min(p, most - (n.prefix_tiles - 1) * p);
    }
  }
  n.merge = args.shared_len || (n.small && !n.whole && own > 32 * kWaves) || n.tile_parts > 1;
  n.planned = q.n_seq > kPlanned && (n.small || n.tiled);
  n.merge_small = !args.shared_len && n.tile_parts <= 1;
  n.merge_rows = (uint32_t)(std::min<uint64_t>(kSmallRows, q.max_q * group) + kWaves - 1) / kWaves;
  return n;
}

// Values and records of a workspace's parts.
struct Room {
  uint64_t prefix, tile, item;  // partial results of a row and head (or of an item's row)
  uint64_t plan, tiles;         // sequences
};

// What a call takes.
Room attn_room(const rlh_kv_pages& kv, const rlh_seqs& q, const rlh_attn_args& args, const Sizes& n) {
  const uint64_t rows = (uint64_t)q.n_rows * args.n_head;
  Room r{};
  r.prefix = args.shared_len ? n.prefix_parts * rows : 0;
  r.tile = n.tiled && (n.tile_parts > 1 || args.shared_len) ? n.tile_parts * rows : 0;
  r.item = n.small && n.merge ? (uint64_t)n.items * kv.n_head_kv * kSmallRows : 0;
  r.plan = n.small ? q.n_seq : 0;
  r.tiles = n.planned && n.tiled ? q.n_seq : 0;
  return r;
}

// What no call with n_seq, n_rows, max_q, max_kv and shared_len up to these
// takes more of. Parts let their tiles' blocks run at once: parts * tiles *
// n_head_kv <= 256, where tiles of 256 rows hold all rows of a KV head, so
// that parts * rows <= 2^16 if there is more than one part (for a last prefix
// tile of up to 128 rows as well: 20 (tiles - 1/2) < 20 tiles - 9).
Room attn_room_within(const rlh_kv_pages& kv, const rlh_seqs& q, const rlh_attn_args& args) {
  const uint64_t group = args.n_head / kv.n_head_kv, rows = (uint64_t)q.n_rows * args.n_head;
  auto divided = [&](uint64_t positions) {  // 0: never
    const uint64_t parts = tile_parts(kv.n_head_kv, positions);
    return parts > 1 ? std::min<uint64_t>(256 * kTileRows, parts * rows) : 0;
  };
  const bool tiled = q.max_q * group > kSmallRows, small = group <= kSmallRows;
  const bool whole = q.max_kv <= kWhole && q.n_seq * kv.n_head_kv <= 256 && (!tiled || q.n_seq == 1);
  Room r{};
  if (args.shared_len) r.prefix = std::max(rows, divided(args.shared_len));
  if (tiled) r.tile = std::max(args.shared_len ? rows : 0, divided(q.max_kv));
  if (small && (args.shared_len || (!whole && q.max_kv > 32 * kWaves)))
    r.item = ((uint64_t)q.n_seq + item_goal(kv.n_head_kv)) * kv.n_head_kv * kSmallRows;
  r.plan = small ? q.n_seq : 0;
  r.tiles = q.n_seq > kPlanned && tiled ? q.n_seq : 0;
  return r;
}

// Places the workspace's parts from `base` on (null: counts only); bytes.
uint64_t place_workspace(Workspace* w, uint8_t* base, uint64_t dim, const Room& r) {
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    uint8_t* p = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  w->prefix_o = (float*)take(r.prefix * dim * 4);
  w->prefix_ml = (float*)take(r.prefix * 8);
  w->tile_o = (float*)take(r.tile * dim * 4);
  w->tile_ml = (float*)take(r.tile * 8);
  w->item_o = (float*)take(r.item * dim * 4);
  w->item_ml = (float*)take(r.item * 8);
  w->plan = (uint32_t*)take(r.plan * 8);
  w->tiles = (uint32_t*)take(r.tiles * 8);
  return at;
}

// The mixed kernels take more LDS than a launch may by default; said once per
// device (idempotent, so two threads may).
template <int D>
constexpr uint32_t kMixedLds = kTileLds<D> > 2 * kSmallLds<D, kWaves> ? kTileLds<D> : 2 * kSmallLds<D, kWaves>;
template <typename T, int D, int MOD>
int allow_lds(int device) {
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_acquire) & bit) return RLH_OK;
  if (hipFuncSetAttribute((const void*)k_attn_mixed<T, D, MOD>, hipFuncAttributeMaxDynamicSharedMemorySize,
                          (int)kMixedLds<D>) != hipSuccess ||
      hipFuncSetAttribute((const void*)k_attn_small<T, D, MOD, kTileWaves>, hipFuncAttributeMaxDynamicSharedMemorySize,
                          (int)kSmallLds<D, kTileWaves>) != hipSuccess) {
    (void)hipGetLastError();
    return serve_error(RLH_EDEVICE, "hipFuncSetAttribute (LDS of the tiled attention kernels)");
  }
  done.fetch_or(bit, std::memory_order_release);
  return RLH_OK;
}

template <typename T, int D, int MOD>
int launch_attn(const Launch& L, int device, hipStream_t s) {
  const uint32_t G = L.a.n_kv;
  const char* what = "rlh_paged_attn";
  if (L.n.planned) RLH_TRY(enqueue(what, k_attn_plan, dim3(1), kPlanThreads, 0, s, L));
  if (L.a.shared_len || L.n.tiled) {
    RLH_TRY((allow_lds<T, D, MOD>(device)));
    const uint32_t blocks = (prefix_blocks(L.n) + L.n.tiles * L.n.tile_parts) * G + (L.n.items * G + 1) / 2;
    RLH_TRY(enqueue(what, k_attn_mixed<T, D, MOD>, dim3(blocks), 64 * kTileWaves, kMixedLds<D>, s, L));
  } else if (L.n.whole) {
    RLH_TRY((allow_lds<T, D, MOD>(device)));
    RLH_TRY(enqueue(what, k_attn_small<T, D, MOD, kTileWaves>, dim3(L.n.items * G), 64 * kTileWaves,
                    kSmallLds<D, kTileWaves>, s, L));
  } else {
    RLH_TRY(enqueue(what, k_attn_small<T, D, MOD, kWaves>, dim3(L.n.items * G), kThreads, kSmallLds<D, kWaves>, s, L));
  }
  if (!L.n.merge) return RLH_OK;
  const uint64_t blocks = L.n.merge_small ? (uint64_t)L.a.b.n_seq * L.n.merge_rows * G
                                          : ((uint64_t)L.a.b.n_rows * L.a.n_head + kWaves - 1) / kWaves;
  return enqueue(what, k_attn_merge<T, D>, dim3((uint32_t)blocks), kThreads, 0, s, L);
}

template <typename T, int D>
int launch_attn(const Launch& L, int mod, int device, hipStream_t s) {
  return mod == kPlain ? launch_attn<T, D, kPlain>(L, device, s)
         : mod == kMod ? launch_attn<T, D, kMod>(L, device, s)
                       : launch_attn<T, D, kWideCap>(L, device, s);
}

template <typename T>
int launch_attn(const Launch& L, uint32_t dim, int mod, int device, hipStream_t s) {
  return dim == 64 ? launch_attn<T, 64>(L, mod, device, s) : launch_attn<T, 128>(L, mod, device, s);
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

uint64_t rlh_paged_attn_workspace(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args) {
  if (check_attn(kv, seqs, args) != RLH_OK || seqs->n_seq == 0 || seqs->n_rows == 0) return 0;
  Workspace w;
  return place_workspace(&w, nullptr, kv->head_dim, attn_room_within(*kv, *seqs, *args));
}

int rlh_paged_attn(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_attn_args* args, void* workspace,
                   uint64_t workspace_bytes, uint32_t* status, void* stream) {
  RLH_TRY(check_attn(kv, seqs, args));
  if (!aligned(status, 4)) return serve_error(RLH_EINVAL, "status is not aligned to 4 bytes");
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  Launch L{};
  L.n = attn_sizes(*kv, *seqs, *args);
  const uint64_t need = place_workspace(&L.ws, (uint8_t*)workspace, kv->head_dim, attn_room(*kv, *seqs, *args, L.n));
  if (need && !workspace) return serve_error(RLH_EINVAL, "workspace is null");
  if (need > workspace_bytes)
    return serve_error(RLH_EINVAL, "workspace of " + std::to_string(workspace_bytes) + " bytes, " + std::to_string(need) + " needed");
  if (need && !aligned(workspace, 16)) return serve_error(RLH_EINVAL, "workspace is not aligned to 16 bytes");
  const uint64_t w = (uint64_t)args->n_head * kv->head_dim;
  if (overlap(workspace, need, args->q, row_bytes_span(seqs->n_rows, args->q_stride, w, 2)) ||
      overlap(workspace, need, args->out, row_bytes_span(seqs->n_rows, args->out_stride, w, 2)) ||
      overlaps_pool(*kv, workspace, need))
    return serve_error(RLH_EINVAL, "workspace overlaps q, out or the pool");
  const uint64_t rows = seqs->n_rows;
  const Area q_start = area_q_start(*seqs), kv_len = area_kv_len(*seqs), table = area_table(*seqs, kv->page_size),
             slopes = area("slopes", args->slopes, args->n_head * 4ull),
             prefix_len = area("prefix_len", args->prefix_len, seqs->n_seq * 4ull),
             shared = area("shared_table", args->shared_len ? args->shared_table : nullptr,
                           args->shared_len / kv->page_size * 4ull),
             st = area("status", status, 4);
  for (const Area& written :
       {Area{"out", args->out, rows, args->out_stride * 2, w * 2}, area("workspace", need ? workspace : nullptr, need)})
    RLH_TRY(check_apart(written, {q_start, kv_len, table, slopes, prefix_len, shared, st}));
  RLH_TRY(check_apart(st, {q_start, kv_len, table, slopes, prefix_len, shared,
                           Area{"q", args->q, rows, args->q_stride * 2, w * 2},
                           area("the pool", kv->k, pool_bytes(*kv)), area("the pool", kv->v, pool_bytes(*kv))}));
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
  p.n_head = args->n_head;
  p.n_kv = kv->n_head_kv;
  p.group = args->n_head / kv->n_head_kv;
  p.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  p.n_pages = (uint32_t)kv->n_pages;
  p.window = args->window;
  p.shared_len = args->shared_len;
  L.a = p;
  L.sc.capped = args->softcap > 0.0f;
  L.sc.mul = score_factor(*args);
  L.sc.cap2 = fminf(args->softcap, kMostCap) * kLog2e;
  L.sc.flip = args->scale < 0.0f ? 0x80008000u : 0u;
  // (a scale of zero, which the exponential could not take in, goes with a bias of zero)
  L.sc.biased = args->slopes || (!L.sc.capped && L.sc.mul == 0.0f);
  const int mod = args->softcap > kNarrowCap ? kWideCap : L.sc.capped || L.sc.biased ? kMod : kPlain;
  if (kv->type == RLH_TYPE_F16) return launch_attn<_Float16>(L, kv->head_dim, mod, dev.device(), (hipStream_t)stream);
  return launch_attn<__bf16>(L, kv->head_dim, mod, dev.device(), (hipStream_t)stream);
}

}  // extern "C"
