"""Plain 64-bit forms of the batched serving operators and the inputs of their
tests: one sequence, one head and one row at a time, from the definitions in
include/rlh_serve.h."""
import math

import numpy as np
import torch

import rlh

TORCH = {rlh.F16: torch.float16, rlh.BF16: torch.bfloat16, rlh.F32: torch.float32}


class Batch:
    """A pool, a ragged batch over it and (new rows, positions) per sequence.
    Pages are handed out in random order; every slot of the pool, also those
    that no sequence holds, is filled with `fill`."""

    def __init__(self, seqs, kv_heads, dim, page, ty, seed=0, shared=0, fill=None, pad_seqs=0, pad_rows=0, extra=2):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.kv_heads, self.dim, self.page, self.ty, self.shared = seqs, kv_heads, dim, page, ty, shared
        counts = [-(-n // page) for _, n in seqs]
        stride = max(counts + [shared // page]) + 1
        own = [max(c - shared // page, 0) for c in counts]
        self.n_pages = sum(own) + shared // page + extra
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table = np.full((len(seqs) + pad_seqs, stride), 0x7ffffff0, np.int64)  # unused entries are no pages
        self.shared_pages = order[:shared // page]
        at = shared // page
        for s, c in enumerate(counts):
            for i in range(shared // page, c):
                table[s, i] = order[at]
                at += 1
        self.table_host = table
        starts = np.cumsum([0] + [q for q, _ in seqs] + [0] * pad_seqs)
        self.n_rows = int(starts[-1]) + pad_rows
        self.n_live = int(starts[-1])
        self.starts = starts
        dt = TORCH[ty]
        shape = (self.n_pages, kv_heads, page, dim)
        if fill is None:
            self.k = torch.randn(shape, generator=g).to(dt).cuda()
            self.v = torch.randn(shape, generator=g).to(dt).cuda()
        else:
            self.k = torch.full(shape, fill, dtype=dt).cuda()
            self.v = torch.full(shape, fill, dtype=dt).cuda()
            for s, (_, n) in enumerate(seqs):
                for j in range(n):
                    p = self.page_of(s, j)
                    self.k[p, :, j % page] = torch.randn((kv_heads, dim), generator=g).to(dt).cuda()
                    self.v[p, :, j % page] = torch.randn((kv_heads, dim), generator=g).to(dt).cuda()
        self.max_q = max([q for q, _ in seqs] + [1])
        self.max_kv = max([n for _, n in seqs] + [self.max_q])
        self.q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        self.kv_len = torch.tensor([n for _, n in seqs] + [12345] * pad_seqs, dtype=torch.int32).cuda()
        self.table = torch.tensor(table, dtype=torch.int32).cuda()
        self.shared_table = torch.tensor(self.shared_pages, dtype=torch.int32).cuda() if shared else None

    def page_of(self, s, j):
        return self.shared_pages[j // self.page] if j < self.shared else int(self.table_host[s, j // self.page])

    def kv(self):
        return rlh.KvPages(self.ty, self.kv_heads, self.dim, self.page, self.n_pages, self.k.data_ptr(),
                           self.v.data_ptr())

    def desc(self):
        return rlh.Seqs(self.table.shape[0], self.n_rows, self.max_q, self.max_kv, self.table.shape[1],
                        self.q_start.data_ptr(), self.kv_len.data_ptr(), self.table.data_ptr())

    def rows_of(self, s):
        """K and V of sequence s in 64 bits: [positions, KV heads, dim]."""
        n = self.seqs[s][1]
        j = np.arange(n)
        pages = torch.tensor([self.page_of(s, int(x)) for x in range(0, n, self.page)], device="cuda")
        pg = pages[torch.tensor(j // self.page, device="cuda")]
        sl = torch.tensor(j % self.page, device="cuda")
        return self.k[pg, :, sl].double(), self.v[pg, :, sl].double()


def attention(b, q, heads, scale, cap=0.0, slopes=None, window=0, prefix=None, hidden_pages=()):
    """(out, bound) in 64 bits. bound: how far a kernel may be off that forms
    scores, maxima and sums in f32, rounds the probabilities to the pool's
    type and rounds the result once, with half = eps / 2 of the type:
      |out| half                       the result's rounding
      sum(p |v|) / L * half            the probabilities' rounding
      sum(p |v|) / L * 2 (ds + n 2^-24)  ds: the largest error of a score (it
         scales p by 1 + ds, once in the sum with v and once in L), n terms
         in f32 sums; a dot of D terms is off by (D + 8) 2^-24 sum |q k|, the
         cap, the bias and the exponent's argument add 8 half steps of their
         own size
      2^-25 sum |v| / L                f16 only: probabilities below 2^-14 are
         rounded to multiples of 2^-24
    where L = sum p with p = exp(s - max s)."""
    group = heads // b.kv_heads
    out = torch.zeros((b.n_rows, heads, b.dim), dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    half = torch.finfo(TORCH[b.ty]).eps / 2
    u = 2.0 ** -24
    for s, (rows, n) in enumerate(b.seqs):
        if rows == 0:
            continue
        k, v = b.rows_of(s)
        r0 = int(b.starts[s])
        i = torch.arange(n - rows, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        see = j <= i
        if window:
            see = see & (j > i - window)
        if prefix is not None:
            see = see | (j < int(prefix[s]))
        gone = torch.tensor([b.page_of(s, x) in hidden_pages for x in range(n)], device="cuda")
        see = see & ~gone[None, :]
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            vh = torch.where(see.any(0)[:, None], vh, 0.0)
            qh = q[r0:r0 + rows, h].double()
            t = scale * (qh @ kh.T)
            ds = (b.dim + 8) * u * abs(scale) * (qh.abs() @ kh.abs().T)
            if cap:
                t = cap * torch.tanh(t / cap)
                ds = ds + 8 * u * cap
            if slopes is not None:
                t = t + float(slopes[h]) * (j - i)
                ds = ds + 8 * u * t.abs()
            ds = ds + 8 * u * t.abs()
            t = torch.where(see, t, -math.inf)
            ds = torch.where(see & torch.isfinite(ds), ds, 0.0).amax(1, keepdim=True)
            top = t.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(t - torch.where(top == -math.inf, 0.0, top)), 0.0)
            L = p.sum(1, keepdim=True)
            L = torch.where(L == 0, 1.0, L)
            o = (p @ vh) / L
            near = (p @ vh.abs()) / L
            e = o.abs() * half + near * (half + 2 * (ds + n * u))
            if b.ty == rlh.F16:
                e = e + 2.0 ** -25 * (see.double() @ vh.abs()) / L
            out[r0:r0 + rows, h], bound[r0:r0 + rows, h] = o, e
    return out, bound


def rotate(x, pos, freqs, magnitude, rot, inter):
    """x [rows, heads, dim] in 64 bits, rotated."""
    x = x.clone()
    a = pos.double()[:, None] * freqs[None, :]
    c, s = (torch.cos(a) * magnitude)[:, None], (torch.sin(a) * magnitude)[:, None]
    lo, hi = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y0, y1 = lo * c - hi * s, hi * c + lo * s
    if inter:
        x[..., 0:rot:2], x[..., 1:rot:2] = y0, y1
    else:
        x[..., :rot // 2], x[..., rot // 2:rot] = y0, y1
    return x


def norm(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def sample(logits, temperature, top_k, top_p, min_p, u):
    """One row, numpy float64, from the definition."""
    x = np.asarray(logits, np.float64)
    n = len(x)
    live = x > -np.inf  # neither NaN nor -inf
    if not live.any():
        return 0
    score = np.where(live, x, -np.inf)
    order = np.argsort(-score, kind="stable")
    top = score[order[0]]
    if not temperature > 0:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(score == top, 1.0, np.exp((score - top) / temperature))
    w = np.where(live & ~np.isnan(w), w, 0.0)
    ws = w[order]
    keep = np.ones(n, bool)
    if 0 < top_k < n:
        keep[top_k:] = False
    if 0 < top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        keep &= (before < np.float32(top_p).astype(np.float64) * ws.sum()) | (np.arange(n) == 0)
    if min_p > 0:
        keep &= ws >= np.float32(min_p).astype(np.float64)
    keep[0] = True
    mass = np.zeros(n)
    mass[order] = np.where(keep, ws, 0.0)
    run = np.cumsum(mass)
    u = float(u)
    u = 0.0 if not u > 0 else u
    hit = np.nonzero(run > u * run[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(mass > 2.0 ** -43)[0][-1])
