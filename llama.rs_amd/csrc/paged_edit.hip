// paged_edit.hip — the paged cache, edited: masks of drafted trees, the branch
// that is kept, the choice of positions that stay, and the move of their rows.
#include <algorithm>

#include "../../include/rlh_cache.h"
#include "paged_device.h"
#include "rlh_device.h"
#include "serve_check.h"

namespace rlh {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)x, lane) | (uint64_t)(uint32_t)__shfl((int)(uint32_t)(x >> 32), lane) << 32;
}

// A value every lane of the wave has.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- trees --------------------------------------------------------------------------

struct TreeParams {
  Batch b;
  const uint32_t *parents, *base;
  uint64_t* masks;
  uint32_t* positions;
  uint32_t* status;
  uint32_t mask_words;
};

// A wave takes a sequence, 64 rows at a time (a block of its own each: it
// waits for nobody). Within them the ancestors are found by doubling: after k
// rounds a lane's bits hold 2^k of them and its pointer the one above; what
// lies before the 64 is the mask of the first ancestor there, complete by then.
// Bound by latency (a round is three exchanges of about 100 cycles): 1.9 us for
// a tree of 26, 2.8 for 120 of up to 63.
__global__ void __launch_bounds__(64) k_tree_masks(TreeParams a) {
  const uint32_t s = blockIdx.x, lane = threadIdx.x;
  bool bad;
  const SeqView v = load_seq(a.b, s, &bad);
  if (bad && lane == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
  if (!v.ok) return;
  const uint32_t base = a.base ? a.base[s] : v.kv_len - v.q_len, words = a.mask_words;
  for (uint32_t c = 0; c * 64 < v.q_len; c++) {
    const uint32_t i = c * 64 + lane;
    uint32_t parent = i < v.q_len ? a.parents[v.q0 + i] : RLH_NO_PARENT;
    if (parent != RLH_NO_PARENT && parent >= i) {
      raise(a.status, RLH_SERVE_BAD_SEQ);
      parent = RLH_NO_PARENT;
    }
    const bool inside = parent != RLH_NO_PARENT && parent >= c * 64;
    uint32_t up = inside ? parent - c * 64 : lane;       // (a lane without one points to itself)
    const uint32_t outside = inside ? RLH_NO_PARENT : parent;
    uint64_t bits = 1ull << lane;
    for (int round = 0; round < 6; round++) {
      bits |= shfl64(bits, (int)up);
      up = (uint32_t)__shfl((int)up, (int)up);
    }
    const uint32_t above = (uint32_t)__shfl((int)outside, (int)up);
    if (i < v.q_len) {
      uint64_t* mask = a.masks + (size_t)(v.q0 + i) * words;
      const uint64_t* from = above != RLH_NO_PARENT ? a.masks + (size_t)(v.q0 + above) * words : nullptr;
      uint32_t depth = (uint32_t)__popcll(bits) - 1;
      for (uint32_t w = 0; w < words; w++) {
        const uint64_t x = w < c ? (from ? from[w] : 0) : w == c ? bits : 0;
        mask[w] = x;
        if (w < c) depth += (uint32_t)__popcll(x);
      }
      if (a.positions) a.positions[v.q0 + i] = base + depth;
    }
    __syncthreads();  // the next rows read these masks
  }
}

struct AcceptParams {
  Batch b;
  rlh_accept_args a;
  uint32_t* status;
};

// A wave takes a sequence; each step asks 64 rows at a time which of them is
// the child, from the kept row on. Bound by latency, two exchanges a step: 2.0 us
// for a tree of 26, 3.8 for 96 of up to 63.
__global__ void __launch_bounds__(64) k_tree_accept(AcceptParams p) {
  const uint32_t s = blockIdx.x, lane = threadIdx.x;
  bool bad;
  const SeqView v = load_seq(p.b, s, &bad);
  if (bad && lane == 0) raise(p.status, RLH_SERVE_BAD_SEQ);
  if (!v.ok) {
    if (lane == 0) p.a.count[s] = 0;
    return;
  }
  const uint32_t *parents = p.a.parents + v.q0, *tokens = p.a.tokens + v.q0, *sampled = p.a.sampled + v.q0;
  uint32_t* path = p.a.path + (size_t)s * p.a.path_stride;
  // the first 64 rows stay in registers
  const bool in0 = lane < v.q_len;
  const uint32_t parent0 = in0 ? parents[lane] : RLH_NO_PARENT, token0 = in0 ? tokens[lane] : 0;
  const uint32_t sampled0 = in0 ? sampled[lane] : 0;
  auto drawn = [&](uint32_t i) {
    return i < 64 ? (uint32_t)__builtin_amdgcn_readlane((int)sampled0, (int)i) : sampled[i];
  };
  uint32_t cur = 0, count = 0, want = drawn(0);
  for (;;) {
    if (lane == 0) path[count] = cur;
    count++;
    uint32_t next = 0;
    for (uint32_t c = cur / 64; c * 64 < v.q_len; c++) {
      const uint32_t i = c * 64 + lane;
      uint32_t parent = parent0, token = token0;
      if (c > 0) {
        parent = i < v.q_len ? parents[i] : RLH_NO_PARENT;
        token = i < v.q_len ? tokens[i] : 0;
      }
      const uint64_t hit = __ballot(i < v.q_len && i > cur && parent == cur && token == want);
      if (hit) {
        next = c * 64 + (uint32_t)__builtin_ctzll(hit);
        break;
      }
    }
    if (next == 0) break;
    cur = next;
    want = drawn(cur);
  }
  if (lane == 0) {
    p.a.count[s] = count;
    p.a.next[s] = want;
    p.a.new_len[s] = v.kv_len - v.q_len + count;
  }
}

// ---- moving rows ----------------------------------------------------------------------

struct MoveParams {
  const uint32_t *kv_len, *table, *index, *count, *base;
  const float* mass;
  float* mass_out;
  void *pool_k, *pool_v;
  uint32_t* status;
  uint32_t n_seq, n_kv, max_kv, table_stride, index_stride, per_head, max_count, page_shift, n_pages;
};

// A block takes a slice of 16 L bytes of the rows of K or V of one KV head of one
// sequence and goes through the list in order, AHEAD rows per thread at a
// time: all of a round's values are read before one of them is written. A row
// comes from its place or from behind it, so what a round writes no later round
// reads; slices have nothing to do with each other. While a round's values are
// on their way the next one's places are looked up. Bound by HBM where there is
// enough to move (24 sequences cut to 2048 of up to 8191: 0.40 GB in 88 us, 4.6
// TB/s; whole rows, four ahead: 164), by rounds for a single one (4096 rows of 8
// heads in 15.7 us, 64 blocks of two rounds each; whole rows: 165).
template <int D, int L, int THREADS, int AHEAD>
__global__ void __launch_bounds__(THREADS) k_paged_move(MoveParams a) {
  constexpr uint32_t kSlices = D / 8 / L, R = THREADS / L;  // rows of a pass
  // the slices of a row go to one XCD (blocks are dealt to the eight in turn), whose L2 holds its lines
  const uint32_t slice = blockIdx.x / 8 % kSlices, of = blockIdx.x / (8 * kSlices) * 8 + blockIdx.x % 8;
  const bool is_v = of & 1;
  const uint32_t h = (of >> 1) % a.n_kv, s = (of >> 1) / a.n_kv;
  if (s >= a.n_seq) return;
  const uint32_t n = a.kv_len[s], count = a.count[s], base = a.base ? a.base[s] : 0;
  if (count == 0) return;
  if (n > a.max_kv || count > a.max_count || base > n || count > n - base) {
    if (threadIdx.x == 0) raise(a.status, RLH_SERVE_BAD_SEQ);
    return;
  }
  const uint32_t* index = a.index + ((size_t)s * (a.per_head ? a.n_kv : 1) + (a.per_head ? h : 0)) * a.index_stride;
  const uint32_t* table = a.table + (size_t)s * a.table_stride;
  const uint32_t c = threadIdx.x % L, r0 = threadIdx.x / L, page_mask = (1u << a.page_shift) - 1;
  u32x4_t* pool = (u32x4_t*)(is_v ? a.pool_v : a.pool_k) + slice * L + c;
  const bool masses = !is_v && slice == 0 && a.mass && c == 0, apart = a.mass != a.mass_out;
  uint32_t at[AHEAD], to[AHEAD];  // rows of the pool (which no memory holds 2^32 of)
  uint32_t what[AHEAD];                // bits: a row, a mass
  // (loads of places that exist, checked afterwards: branches would put them one behind the other)
  auto look_up = [&](uint32_t j0) {
    uint32_t from[AHEAD], ps[AHEAD], pd[AHEAD], bad = 0;
#pragma unroll
    for (int u = 0; u < AHEAD; u++) from[u] = index[min(j0 + u * R + r0, count - 1)];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      ps[u] = table[(base + min(from[u], n - base - 1)) >> a.page_shift];
      pd[u] = table[(base + min(j0 + u * R + r0, count - 1)) >> a.page_shift];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const uint32_t j = j0 + u * R + r0;
      const bool any = j < count && (from[u] != j || (masses && apart)), fits = from[u] >= j && from[u] < n - base;
      const bool exist = ps[u] < a.n_pages && pd[u] < a.n_pages, ok = any && fits && exist;
      bad |= (any && !fits ? RLH_SERVE_BAD_SEQ : 0u) | (any && fits && !exist ? RLH_SERVE_BAD_PAGE : 0u);
      at[u] = ok ? ((ps[u] * a.n_kv + h) << a.page_shift) + ((base + from[u]) & page_mask) : 0;
      to[u] = ok ? ((pd[u] * a.n_kv + h) << a.page_shift) + ((base + j) & page_mask) : 0;
      what[u] = ok ? (from[u] != j ? 1u : 0u) | (masses ? 2u : 0u) : 0u;
    }
    if (bad && c == 0) raise(a.status, bad);
  };
  look_up(0);
  for (uint32_t j0 = 0; j0 < count; j0 += R * AHEAD) {
    u32x4_t row[AHEAD];
    float mass[AHEAD];
    uint32_t dst[AHEAD], moves[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      if (__ballot(what[u] & 1)) row[u] = pool[(size_t)at[u] * (D / 8)];
      dst[u] = to[u];
      moves[u] = what[u];
    }
    if (masses) {
#pragma unroll
      for (int u = 0; u < AHEAD; u++) mass[u] = a.mass[at[u]];
    }
    if (j0 + R * AHEAD < count) look_up(j0 + R * AHEAD);
    wait_vmcnt<0>();  // the values have arrived: another wave may write where they were
    __syncthreads();
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
      if (moves[u] & 1) pool[(size_t)dst[u] * (D / 8)] = row[u];
    if (masses) {
#pragma unroll
      for (int u = 0; u < AHEAD; u++)
        if (moves[u] & 2) a.mass_out[dst[u]] = mass[u];
    }
  }
}

template <int D, int L, int THREADS, int AHEAD>
int launch_move(const MoveParams& p, hipStream_t stream) {
  const uint32_t of = (p.n_seq * p.n_kv * 2 + 7) / 8 * 8;
  return enqueue("rlh_paged_move", k_paged_move<D, L, THREADS, AHEAD>, dim3(of * (D / 8 / L)), THREADS, 0, stream, p);
}
template <int D>
int launch_move(const MoveParams& p, hipStream_t stream) {
  // Short lists (accepted branches): whole rows by small blocks, one row ahead (three
  // rows of 96 sequences: 3.7 us, by the other form 7.7). Long ones: slices of 64 bytes,
  // while a launch holds them (fewer than 2^32 threads): 2^18 lists fill the card without.
  if (p.max_count <= 256 || (uint64_t)p.n_seq * p.n_kv > (1u << 18)) return launch_move<D, D / 8, 256, 1>(p, stream);
  return launch_move<D, 4, 1024, 8>(p, stream);
}

// ---- what stays -------------------------------------------------------------------------

struct EvictParams {
  const uint32_t *kv_len, *table;
  const float* mass;
  uint32_t *keep, *count;
  uint32_t* status;
  uint32_t n_kv, max_kv, table_stride, page_shift, n_pages, budget, first, last, keep_stride;
};

// Masses as whole numbers of the same order; 0: no position, 1: NaN.
__device__ __forceinline__ uint32_t mass_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as 0
  return x != x ? 1u : b >> 31 ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKeptKey = 0xffffffffu;  // above every mass

// How many lanes below this one are in the mask.
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kEvictBits[3] = {13, 10, 9};  // of a key, from the top
constexpr int kEvictBins = 1 << 13;

// A block takes one KV head of one sequence. The smallest kept key is found
// from three histograms of 13, 10 and 9 of its bits; then each wave counts the
// larger and the equal ones of its stretch and lists those that stay. With up
// to 1024 R positions the keys stay in registers (R = 0: read anew each time).
// Bound by one CU's instructions, LDS counters among them: 30 us for 40000
// positions (95 with keys read anew, 33 with bits 11, 11 and 10, whose first
// counters collide more), 11 for 192 lists of about 5000.
template <int R>
__global__ void __launch_bounds__(kEvictThreads) k_evict_select(EvictParams a) {
  __shared__ uint32_t bins[kEvictBins];
  __shared__ uint32_t sums[2][kEvictWaves];
  __shared__ uint32_t found[2];
  const uint32_t h = blockIdx.x % a.n_kv, s = blockIdx.x / a.n_kv;
  const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const uint32_t n = a.kv_len[s];
  if (n > a.max_kv) {
    if (t == 0 && h == 0) {
      raise(a.status, RLH_SERVE_BAD_SEQ);
      a.count[s] = 0;
    }
    return;
  }
  if (t == 0 && h == 0) a.count[s] = min(n, a.budget);
  uint32_t* keep = a.keep + ((size_t)s * a.n_kv + h) * a.keep_stride;
  if (n <= a.budget) {
    for (uint32_t j = t; j < n; j += kEvictThreads) keep[j] = j;
    return;
  }
  const uint32_t* table = a.table + (size_t)s * a.table_stride;
  auto key_of = [&](uint32_t j) -> uint32_t {
    if (j >= n) return 0u;
    if (j < a.first || j >= n - a.last) return kKeptKey;
    const uint32_t page = table[j >> a.page_shift];
    if (page >= a.n_pages) {
      raise(a.status, RLH_SERVE_BAD_PAGE);
      return 1u;
    }
    return mass_key(a.mass[(((size_t)page * a.n_kv + h) << a.page_shift) + (j & ((1u << a.page_shift) - 1))]);
  };
  // each wave's stretch, 64 positions at a time
  const uint32_t rounds = (n + kEvictThreads - 1) / kEvictThreads;
  const uint32_t j0 = wave * rounds * 64 + lane;
  uint32_t keys[R ? R : 1];
  // f(position, key) for the wave's positions in order
  auto each = [&](auto f) {
    if constexpr (R != 0) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        if ((uint32_t)r >= rounds) continue;
        asm volatile("" : "+v"(keys[r]));  // (no comparison is kept from one sweep for the next)
        f(j0 + r * 64, keys[r]);
      }
    } else {
      for (uint32_t r = 0; r < rounds; r++) f(j0 + r * 64, key_of(j0 + r * 64));
    }
  };
  if constexpr (R != 0) {
    // pages, then masses, kAtOnce at a time: what is not a mass is read from the sequence's first place
    // (a branch among them would put one load behind the other)
    bool missing = false;
    constexpr int kAtOnce = R < 20 ? R : 20;
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += kAtOnce) {
      uint32_t page[kAtOnce];
#pragma unroll
      for (int r = 0; r < kAtOnce; r++) {
        const uint32_t j = j0 + (r0 + r) * 64;
        page[r] = table[(j < n ? j : 0u) >> a.page_shift];
      }
      float x[kAtOnce];
#pragma unroll
      for (int r = 0; r < kAtOnce; r++) {
        const uint32_t slot = (j0 + (r0 + r) * 64) & ((1u << a.page_shift) - 1);
        x[r] = a.mass[(((size_t)(page[r] < a.n_pages ? page[r] : 0u) * a.n_kv + h) << a.page_shift) + slot];
      }
#pragma unroll
      for (int r = 0; r < kAtOnce; r++) {
        asm volatile("" : "+v"(x[r]));  // (or the load would move behind the conditions below)
        const uint32_t j = j0 + (r0 + r) * 64;
        const bool middle = j >= a.first && j < n - a.last, exists = page[r] < a.n_pages;
        missing |= middle && !exists;
        keys[r0 + r] = j >= n ? 0u : !middle ? kKeptKey : !exists ? 1u : mass_key(x[r]);
      }
    }
    if (missing) raise(a.status, RLH_SERVE_BAD_PAGE);
  }
  uint32_t prefix = 0, left = a.budget;  // keys that begin with `prefix`: so many of them stay
#pragma unroll
  for (int pass = 0; pass < 3; pass++) {
    const int width = kEvictBits[pass], shift = pass == 0 ? 32 - width : pass == 1 ? kEvictBits[2] : 0;
    const int kMine = pass == 0 ? kEvictBins / kEvictThreads : 1;  // bins of a thread
    for (uint32_t b = t; b < 1u << width; b += kEvictThreads) bins[b] = 0;
    __syncthreads();
    each([&](uint32_t, uint32_t k) {
      if (pass != 0 && k >> (shift + width) != prefix) return;
      const uint32_t bin = k >> shift & ((1u << width) - 1);
      // (lanes of one bin would take turns at it: where all are, one counts for them)
      const uint32_t bin0 = uniform(bin);
      const uint64_t here = __ballot(true);
      if (__ballot(bin == bin0) != here)
        atomicAdd(&bins[bin], 1u);
      else if (lane == (uint32_t)__builtin_ctzll(here))
        atomicAdd(&bins[bin], (uint32_t)__popcll(here));
    });
    __syncthreads();
    // from the top: the bin in which the count passes what is left
    uint32_t mine[kEvictBins / kEvictThreads], sum = 0;
#pragma unroll
    for (int i = 0; i < kMine; i++) {
      const uint32_t b = t * kMine + i;
      mine[i] = b < 1u << width ? bins[(1u << width) - 1 - b] : 0;
      sum += mine[i];
    }
    uint32_t upto = wave_scan(sum);
    if (lane == 63) sums[0][wave] = upto;
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) upto += sums[0][w];
    uint32_t before = upto - sum;
    if (before < left && upto >= left) {
#pragma unroll
      for (int i = 0; i < kMine; i++) {
        if (before < left && before + mine[i] >= left) {
          found[0] = (1u << width) - 1 - (t * kMine + i);
          found[1] = left - before;
        }
        before += mine[i];
      }
    }
    __syncthreads();
    prefix = prefix << width | found[0];
    left = found[1];
    __syncthreads();
  }
  // `prefix` is the smallest key that stays, of `left` positions
  uint32_t above = 0, equal = 0;
  each([&](uint32_t, uint32_t k) {
    above += (uint32_t)__popcll(__ballot(k > prefix));
    equal += (uint32_t)__popcll(__ballot(k == prefix));
  });
  if (lane == 0) {
    sums[0][wave] = above;
    sums[1][wave] = equal;
  }
  __syncthreads();
  uint32_t at = 0, ties = 0, all_ties = 0;
  for (uint32_t w = 0; w < kEvictWaves; w++) {
    at += w < wave ? sums[0][w] : 0u;
    ties += w < wave ? sums[1][w] : 0u;
    all_ties += sums[1][w];
  }
  at += min(ties, left);
  if (all_ties == left) {
    each([&](uint32_t j, uint32_t k) {
      const uint64_t all = __ballot(k >= prefix);
      if (k >= prefix) keep[at + lanes_below(all)] = j;
      at += (uint32_t)__popcll(all);
    });
  } else {
    each([&](uint32_t j, uint32_t k) {
      const uint64_t same = __ballot(k == prefix);
      const bool stays = k > prefix || (k == prefix && ties + lanes_below(same) < left);
      const uint64_t all = __ballot(stays);
      if (stays) keep[at + lanes_below(all)] = j;
      at += (uint32_t)__popcll(all);
      ties += (uint32_t)__popcll(same);
    });
  }
}

// ---- checks -----------------------------------------------------------------------------

// The batch's rows, for entries that touch no pages. (No device needed.)
int check_nodes(const rlh_seqs* seqs) {
  if (!seqs) return serve_error(RLH_EINVAL, "null argument");
  if (seqs->n_seq > 65535) return serve_error(RLH_EUNSUP, "more than 65535 sequences");
  if (seqs->n_rows > 0x800000u) return serve_error(RLH_EUNSUP, "more than 2^23 rows");
  if (seqs->n_seq == 0) return RLH_OK;
  if (seqs->n_rows != 0) {
    if (seqs->max_q == 0 || seqs->max_q > seqs->n_rows) return serve_error(RLH_EINVAL, "max_q outside [1, n_rows]");
    if (seqs->max_kv < seqs->max_q) return serve_error(RLH_EINVAL, "max_kv below max_q");
    if (seqs->max_kv >= (1u << 30)) return serve_error(RLH_EUNSUP, "max_kv of 2^30 or more");
  }
  if (!seqs->q_start || !seqs->kv_len) return serve_error(RLH_EINVAL, "a batch array is null");
  if (!aligned(seqs->q_start, 4) || !aligned(seqs->kv_len, 4))
    return serve_error(RLH_EINVAL, "a batch array is not aligned to 4 bytes");
  return RLH_OK;
}

// The pool and the batch's lengths and pages, for entries without rows.
int check_cached(const rlh_kv_pages* kv, const rlh_seqs* seqs) {
  if (!kv || !seqs) return serve_error(RLH_EINVAL, "null argument");
  rlh_seqs s = *seqs;
  s.n_rows = s.max_q = 1;
  s.q_start = s.kv_len;
  if (s.max_kv == 0) {  // all sequences are empty
    s.max_kv = 1;
    s.table_stride = std::max(s.table_stride, 1u);
  }
  return check_batch(kv, &s, kv->n_head_kv);
}

// Words that a call reads or writes: present and aligned.
int check_words(const char* name, const void* p) {
  if (!p) return serve_error(RLH_EINVAL, std::string(name) + " is null");
  if (!aligned(p, 4)) return serve_error(RLH_EINVAL, std::string(name) + " is not aligned to 4 bytes");
  return RLH_OK;
}

Area area_mass(const char* name, const rlh_kv_pages& kv, const float* mass) {
  return area(name, mass, kv.n_pages * kv.n_head_kv * kv.page_size * 4);
}

}  // namespace
}  // namespace rlh

using namespace rlh;

extern "C" {

int rlh_tree_masks(const rlh_seqs* seqs, const uint32_t* parents, const uint32_t* base, uint64_t* masks,
                   uint32_t mask_words, uint32_t* positions, uint32_t* status, void* stream) {
  RLH_TRY(check_nodes(seqs));
  if (seqs->n_seq == 0 || seqs->n_rows == 0) return RLH_OK;
  RLH_TRY(check_words("parents", parents));
  if (!masks || !aligned(masks, 8)) return serve_error(RLH_EINVAL, "masks is null or not aligned to 8 bytes");
  if ((uint64_t)mask_words * 64 < seqs->max_q) return serve_error(RLH_EINVAL, "mask_words holds fewer than max_q bits");
  const uint64_t n = seqs->n_rows;
  if (n * mask_words > (1ull << 32)) return serve_error(RLH_EUNSUP, "n_rows * mask_words above 2^32");
  if (!aligned(base, 4) || !aligned(positions, 4) || !aligned(status, 4))
    return serve_error(RLH_EINVAL, "base, positions or status is not aligned to 4 bytes");
  const Area q_start = area_q_start(*seqs), kv_len = area_kv_len(*seqs), up = area("parents", parents, n * 4),
             from = area("base", base, seqs->n_seq * 4ull), bits = area("masks", masks, n * mask_words * 8),
             pos = area("positions", positions, n * 4), st = area("status", status, 4);
  RLH_TRY(check_apart(bits, {q_start, kv_len, up, from, pos, st}));
  RLH_TRY(check_apart(pos, {q_start, kv_len, up, from, st}));
  RLH_TRY(check_apart(st, {q_start, kv_len, up, from}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("q_start", seqs->q_start));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("parents", parents));
  RLH_TRY(dev("base", base));
  RLH_TRY(dev("masks", masks));
  RLH_TRY(dev("positions", positions));
  RLH_TRY(dev("status", status));
  TreeParams p{};
  p.b = Batch{seqs->n_seq, seqs->n_rows, seqs->max_q, seqs->max_kv, 0, seqs->q_start, seqs->kv_len, nullptr};
  p.parents = parents;
  p.base = base;
  p.masks = masks;
  p.positions = positions;
  p.status = status;
  p.mask_words = mask_words;
  return enqueue("rlh_tree_masks", k_tree_masks, dim3(seqs->n_seq), 64, 0, (hipStream_t)stream, p);
}

int rlh_tree_accept(const rlh_seqs* seqs, const rlh_accept_args* args, uint32_t* status, void* stream) {
  if (!args) return serve_error(RLH_EINVAL, "null argument");
  RLH_TRY(check_nodes(seqs));
  if (seqs->n_seq == 0) return RLH_OK;
  const uint64_t n = seqs->n_rows, seqs_n = seqs->n_seq;
  if (n) {
    RLH_TRY(check_words("parents", args->parents));
    RLH_TRY(check_words("tokens", args->tokens));
    RLH_TRY(check_words("sampled", args->sampled));
    RLH_TRY(check_words("path", args->path));
    if (args->path_stride < seqs->max_q) return serve_error(RLH_EINVAL, "path_stride below max_q");
  }
  RLH_TRY(check_words("count", args->count));
  RLH_TRY(check_words("next", args->next));
  RLH_TRY(check_words("new_len", args->new_len));
  if (!aligned(status, 4)) return serve_error(RLH_EINVAL, "status is not aligned to 4 bytes");
  const Area q_start = area_q_start(*seqs), kv_len = area_kv_len(*seqs), up = area("parents", args->parents, n * 4),
             tokens = area("tokens", args->tokens, n * 4), sampled = area("sampled", args->sampled, n * 4),
             path{"path", n ? args->path : nullptr, seqs_n, args->path_stride * 4ull, seqs->max_q * 4ull},
             count = area("count", args->count, seqs_n * 4), next = area("next", args->next, seqs_n * 4),
             new_len = area("new_len", args->new_len, seqs_n * 4), st = area("status", status, 4);
  RLH_TRY(check_apart(path, {q_start, kv_len, up, tokens, sampled, count, next, new_len, st}));
  RLH_TRY(check_apart(count, {q_start, kv_len, up, tokens, sampled, next, new_len, st}));
  RLH_TRY(check_apart(next, {q_start, kv_len, up, tokens, sampled, new_len, st}));
  RLH_TRY(check_apart(new_len, {q_start, kv_len, up, tokens, sampled, st}));
  RLH_TRY(check_apart(st, {q_start, kv_len, up, tokens, sampled}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("q_start", seqs->q_start));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  if (n) {
    RLH_TRY(dev("parents", args->parents));
    RLH_TRY(dev("tokens", args->tokens));
    RLH_TRY(dev("sampled", args->sampled));
    RLH_TRY(dev("path", args->path));
  }
  RLH_TRY(dev("count", args->count));
  RLH_TRY(dev("next", args->next));
  RLH_TRY(dev("new_len", args->new_len));
  RLH_TRY(dev("status", status));
  AcceptParams p{};
  p.b = Batch{seqs->n_seq, seqs->n_rows, seqs->max_q, seqs->max_kv, 0, seqs->q_start, seqs->kv_len, nullptr};
  p.a = *args;
  p.status = status;
  return enqueue("rlh_tree_accept", k_tree_accept, dim3(seqs->n_seq), 64, 0, (hipStream_t)stream, p);
}

int rlh_paged_move(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_move_args* args, uint32_t* status,
                   void* stream) {
  if (!args) return serve_error(RLH_EINVAL, "null argument");
  RLH_TRY(check_cached(kv, seqs));
  if (seqs->n_seq == 0 || args->max_count == 0) return RLH_OK;
  RLH_TRY(check_words("index", args->index));
  RLH_TRY(check_words("count", args->count));
  if (args->max_count > args->index_stride) return serve_error(RLH_EINVAL, "max_count above index_stride");
  if (!args->mass != !args->mass_out) return serve_error(RLH_EINVAL, "one of mass and mass_out is null");
  if (!aligned(args->base, 4) || !aligned(args->mass, 4) || !aligned(args->mass_out, 4) || !aligned(status, 4))
    return serve_error(RLH_EINVAL, "base, mass, mass_out or status is not aligned to 4 bytes");
  const uint64_t lists = (uint64_t)seqs->n_seq * (args->per_head ? kv->n_head_kv : 1);
  const Area kv_len = area_kv_len(*seqs), table = area_table(*seqs, kv->page_size),
             index{"index", args->index, lists, args->index_stride * 4ull, args->max_count * 4ull},
             count = area("count", args->count, seqs->n_seq * 4ull), base = area("base", args->base, seqs->n_seq * 4ull),
             mass = area_mass("mass", *kv, args->mass), mass_out = area_mass("mass_out", *kv, args->mass_out),
             st = area("status", status, 4), pool_k = area("the pool", kv->k, pool_bytes(*kv)),
             pool_v = area("the pool", kv->v, pool_bytes(*kv));
  for (const Area& written : {pool_k, pool_v, mass_out, st}) RLH_TRY(check_apart(written, {kv_len, table, index, count, base}));
  for (const Area& pool : {pool_k, pool_v}) RLH_TRY(check_apart(pool, {mass, mass_out, st}));
  RLH_TRY(check_apart(st, {mass, mass_out}));
  if (args->mass != args->mass_out) RLH_TRY(check_apart(mass_out, {mass}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("k pages", kv->k));
  RLH_TRY(dev("v pages", kv->v));
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("table", seqs->table));
  RLH_TRY(dev("index", args->index));
  RLH_TRY(dev("count", args->count));
  RLH_TRY(dev("base", args->base));
  RLH_TRY(dev("mass", args->mass));
  RLH_TRY(dev("mass_out", args->mass_out));
  RLH_TRY(dev("status", status));
  MoveParams p{};
  p.kv_len = seqs->kv_len;
  p.table = seqs->table;
  p.index = args->index;
  p.count = args->count;
  p.base = args->base;
  p.mass = args->mass;
  p.mass_out = args->mass_out;
  p.pool_k = kv->k;
  p.pool_v = kv->v;
  p.status = status;
  p.n_seq = seqs->n_seq;
  p.n_kv = kv->n_head_kv;
  p.max_kv = seqs->max_kv;
  p.table_stride = seqs->table_stride;
  p.index_stride = args->index_stride;
  p.per_head = args->per_head;
  p.max_count = args->max_count;
  p.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  p.n_pages = (uint32_t)kv->n_pages;
  return kv->head_dim == 64 ? launch_move<64>(p, (hipStream_t)stream) : launch_move<128>(p, (hipStream_t)stream);
}

int rlh_evict_select(const rlh_kv_pages* kv, const rlh_seqs* seqs, const rlh_evict_args* args, uint32_t* status,
                     void* stream) {
  if (!args) return serve_error(RLH_EINVAL, "null argument");
  RLH_TRY(check_cached(kv, seqs));
  if (args->budget == 0) return serve_error(RLH_EINVAL, "budget is 0");
  if ((uint64_t)args->first_kept + args->last_kept > args->budget)
    return serve_error(RLH_EINVAL, "first_kept + last_kept above budget");
  if (seqs->n_seq == 0) return RLH_OK;
  const uint32_t most = std::min(args->budget, seqs->max_kv);
  RLH_TRY(check_words("mass", args->mass));
  RLH_TRY(check_words("keep", args->keep));
  RLH_TRY(check_words("count", args->count));
  if (args->keep_stride < most) return serve_error(RLH_EINVAL, "keep_stride below min(budget, max_kv)");
  if (!aligned(status, 4)) return serve_error(RLH_EINVAL, "status is not aligned to 4 bytes");
  const Area kv_len = area_kv_len(*seqs), table = area_table(*seqs, kv->page_size),
             mass = area_mass("mass", *kv, args->mass), count = area("count", args->count, seqs->n_seq * 4ull),
             keep{"keep", args->keep, (uint64_t)seqs->n_seq * kv->n_head_kv, args->keep_stride * 4ull, most * 4ull},
             st = area("status", status, 4);
  RLH_TRY(check_apart(keep, {kv_len, table, mass, count, st}));
  RLH_TRY(check_apart(count, {kv_len, table, mass, st}));
  RLH_TRY(check_apart(st, {kv_len, table, mass}));
  DeviceCheck dev;
  RLH_TRY(dev.begin());
  RLH_TRY(dev("kv_len", seqs->kv_len));
  RLH_TRY(dev("table", seqs->table));
  RLH_TRY(dev("mass", args->mass));
  RLH_TRY(dev("keep", args->keep));
  RLH_TRY(dev("count", args->count));
  RLH_TRY(dev("status", status));
  EvictParams p{};
  p.kv_len = seqs->kv_len;
  p.table = seqs->table;
  p.mass = args->mass;
  p.keep = args->keep;
  p.count = args->count;
  p.status = status;
  p.n_kv = kv->n_head_kv;
  p.max_kv = seqs->max_kv;
  p.table_stride = seqs->table_stride;
  p.page_shift = (uint32_t)__builtin_ctz(kv->page_size);
  p.n_pages = (uint32_t)kv->n_pages;
  p.budget = args->budget;
  p.first = args->first_kept;
  p.last = args->last_kept;
  p.keep_stride = args->keep_stride;
  const uint32_t rounds = (seqs->max_kv + kEvictThreads - 1) / kEvictThreads;
  const auto kernel = rounds <= 8 ? k_evict_select<8> : rounds <= 16 ? k_evict_select<16>
                      : rounds <= 40 ? k_evict_select<40> : k_evict_select<0>;
  return enqueue("rlh_evict_select", kernel, dim3(seqs->n_seq * kv->n_head_kv), kEvictThreads, 0, (hipStream_t)stream, p);
}

}  // extern "C"
