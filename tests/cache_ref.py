"""Plain 64-bit forms of the operators that edit a paged cache, from the
definitions in include/rlh_cache.h, and the inputs of their tests."""
import math
import random

import numpy as np
import torch

import rlh
import serve_ref as ref

U = 2.0 ** -24


def random_tree(rng, n, reach=9, roots=0.0):
    """Parents of n nodes; the first has none, others none with `roots`."""
    return [rlh.NO_PARENT if i == 0 or rng.random() < roots else rng.randrange(max(0, i - reach), i) for i in range(n)]


def lineage(parents, i):
    """A node and its ancestors, by walking up; a parent that is not smaller
    is none."""
    line = [i]
    while parents[i] < i:
        i = parents[i]
        line.append(i)
    return line


def mask_matrix(parents):
    see = np.zeros((len(parents), len(parents)), bool)
    for i in range(len(parents)):
        see[i, lineage(parents, i)] = True
    return see


def pack(see, words):
    """Rows of truth values as words of 64 bits (int64 tensors hold them)."""
    rows, n = see.shape
    bits = np.zeros((rows, words * 64), np.uint8)
    bits[:, :n] = see
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64)


def tree_sees(see, first, window):
    """[row, position] of a sequence: what its drafted rows see."""
    rows = see.shape[0]
    out = np.zeros((rows, first + rows), bool)
    for i in range(rows):
        low = max(0, first + int(see[i].sum()) - window) if window else 0
        out[i, min(low, first):first] = True
        out[i, first:] = see[i]
    return out


def causal_sees(rows, n, window=0, prefix=0):
    i, j = np.arange(n - rows, n)[:, None], np.arange(n)[None, :]
    see = j <= i
    if window:
        see &= j > i - window
    return see | (j < prefix)


def scores(b, s, q, h, heads, scale, cap=0.0, slope=0.0):
    """Scores of sequence s and query head h in 64 bits, and how far f32 may
    be off: a dot of D terms (D + 8) 2^-24 sum |q k|, the cap, the bias and the
    exponent's argument 8 half steps of their own size."""
    rows, n = b.seqs[s]
    k, _ = b.rows_of(s)
    kh = k[:, h // (heads // b.kv_heads)]
    r0 = int(b.starts[s])
    qh = q[r0:r0 + rows, h].double()
    t = scale * (qh @ kh.T)
    off = (b.dim + 8) * U * abs(scale) * (qh.abs() @ kh.abs().T)
    if cap:
        t = cap * torch.tanh(t / cap)
        off = off + 8 * U * cap
    if slope:
        i = torch.arange(n - rows, n, device="cuda")[:, None]
        t = t + slope * (torch.arange(n, device="cuda")[None, :] - i)
    return t, off + 8 * U * t.abs()


def attention(b, q, heads, sees, scale, cap=0.0, slopes=None):
    """(out, its bound, lse, its bound) in 64 bits, where sees[s] says which
    positions the rows of sequence s see. The bound of out is that of
    serve_ref.attention; that of lse: the scores', n terms of a sum, and its
    own arithmetic (8 half steps of the sizes in it)."""
    shape = (b.n_rows, heads, b.dim)
    out, bound = (torch.zeros(shape, dtype=torch.float64, device="cuda") for _ in range(2))
    lse, far = (torch.zeros(shape[:2], dtype=torch.float64, device="cuda") for _ in range(2))
    half = torch.finfo(ref.TORCH[b.ty]).eps / 2
    for s, (rows, n) in enumerate(b.seqs):
        if rows == 0:
            continue
        see = torch.tensor(sees[s], device="cuda")
        _, v = b.rows_of(s)
        r0 = int(b.starts[s])
        for h in range(heads):
            t, ds = scores(b, s, q, h, heads, scale, cap, float(slopes[h]) if slopes is not None else 0.0)
            vh = torch.where(see.any(0)[:, None], v[:, h // (heads // b.kv_heads)], 0.0)
            t = torch.where(see, t, -math.inf)
            ds = torch.where(see & torch.isfinite(ds), ds, 0.0).amax(1, keepdim=True)
            top = t.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.where(see, torch.exp(t - top), 0.0)
            total = p.sum(1, keepdim=True)
            L = torch.where(total == 0, 1.0, total)
            o, near = (p @ vh) / L, (p @ vh.abs()) / L
            e = o.abs() * half + near * (half + 2 * (ds + n * U))
            if b.ty == rlh.F16:
                e = e + 2.0 ** -25 * (see.double() @ vh.abs()) / L
            out[r0:r0 + rows, h], bound[r0:r0 + rows, h] = o, e
            ls = (top + torch.log(total))[:, 0]
            lse[r0:r0 + rows, h] = ls
            far[r0:r0 + rows, h] = ds[:, 0] + n * U + 8 * U * (ls.abs() + top[:, 0].abs() + math.log2(n + 1) + 8)
    return out, bound, lse, far


def mass(b, q, heads, sees, lse, scale, decay, old, cap=0.0, slopes=None, shared=0):
    """(mass, its bound): a weight is off by its score's error and 8 half steps
    of the sizes in the exponent, a sum of R terms by R half steps."""
    group = heads // b.kv_heads
    got, bound = old.double(), torch.zeros(old.shape, dtype=torch.float64, device="cuda")
    for s, (rows, n) in enumerate(b.seqs):
        if rows == 0:
            continue
        see = torch.tensor(sees[s], device="cuda")
        r0 = int(b.starts[s])
        j = torch.arange(shared, n, device="cuda")
        pages = torch.tensor([b.page_of(s, int(x)) for x in range(shared, n, b.page)], device="cuda")[(j - shared) // b.page]
        for g in range(b.kv_heads):
            add, off = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
            for h in range(g * group, (g + 1) * group):
                t, ds = scores(b, s, q, h, heads, scale, cap, float(slopes[h]) if slopes is not None else 0.0)
                ls = lse[r0:r0 + rows, h].double()[:, None]
                p = torch.where(see & (ls > -math.inf), torch.exp(t - ls), 0.0)
                rel = torch.where(p > 0, ds + 8 * U * (t.abs() + ls.abs() + 1), 0.0)
                add += p.sum(0)
                off += (p * rel).sum(0)
            was = old[pages, g, j % b.page].double()
            was = torch.where(j < n - rows, decay * was, 0.0) if decay else torch.zeros_like(was)
            got[pages, g, j % b.page] = was + add[shared:]
            bound[pages, g, j % b.page] = off[shared:] + (rows * group + 4) * U * add[shared:] + 4 * U * was.abs() + 2.0 ** -140
    return got, bound


def evict(mass_row, budget, first, last):
    """Kept positions of one sequence and head: numpy, ascending."""
    n = len(mass_row)
    if n <= budget:
        return np.arange(n)
    kept = set(range(first)) | set(range(n - last, n))
    middle = [j for j in range(first, n - last)]
    worth = [-math.inf if np.isnan(x) else float(x) for x in mass_row]
    order = sorted(middle, key=lambda j: (np.isnan(mass_row[j]), -worth[j] + 0.0, j))
    return np.array(sorted(kept | set(order[:budget - first - last])))


def accept(parents, tokens, sampled):
    """Numbers of the kept nodes, by walking."""
    path = [0]
    while True:
        r = path[-1]
        child = next((c for c in range(r + 1, len(parents)) if parents[c] == r and tokens[c] == sampled[r]), None)
        if child is None:
            return path
        path.append(child)


def rng(seed):
    return random.Random(seed)
