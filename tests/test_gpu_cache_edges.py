"""The operators that edit a paged cache (include/rlh_cache.h) where their
kernels go on for long or reach a limit, against the 64-bit forms of
tests/cache_ref.py."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import rlh
import serve_ref as ref
from test_gpu_cache import at, check_tree, run_move, run_tree, stream, tree_case, word

pytestmark = pytest.mark.gpu


# ---- moving rows ------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
def test_move_of_more_lists_than_slices_fit(dim):
    """65535 sequences of 32 KV heads, lists past 256 entries: a launch of slices
    would hold 2^32 threads. Three sequences have rows to move."""
    n, kv, live = 65535, 32, (0, 40001, 65534)
    lengths = [300 if s in live else 0 for s in range(n)]
    b = ref.Batch([(0, x) for x in lengths], kv, dim, 16, rlh.F16, seed=dim, pad_rows=1)
    r = np.random.default_rng(dim)
    index, count = np.zeros((n, 1, 260), np.int32), np.zeros(n, np.int64)
    for s in live:
        index[s, 0] = np.sort(r.choice(300, 260, replace=False))
        count[s] = 260
    k, v = b.k.clone(), b.v.clone()
    for s in live:
        src, dst = index[s, 0], np.arange(260)
        for old, new in ((b.k, k), (b.v, v)):
            new[[b.page_of(s, j) for j in dst], :, dst % 16] = old[[b.page_of(s, int(j)) for j in src], :, src % 16]
    st = word()
    run_move(b, index, count, per_head=False, status=st, max_count=260)
    assert int(st) == 0
    assert torch.equal(b.k, k) and torch.equal(b.v, v)


# ---- windows that bound the drafts ----------------------------------------------------

WINDOWED = {
    "few rows": dict(seqs=[(4, 300), (3, 3), (2, 65), (4, 6)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, window=2),
    "few rows, many": dict(seqs=[(1 + i % 4, 5 + (i * 37) % 300) for i in range(270)], heads=4, kv=1, dim=64, page=32,
                           ty=rlh.BF16, window=3),
    "one token": dict(seqs=[(40, 500), (1, 300), (70, 70)], heads=8, kv=2, dim=64, page=16, ty=rlh.BF16, window=1),
    "deep": dict(seqs=[(130, 900), (64, 64), (65, 100), (3, 40)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, window=33),
    "near the depth": dict(seqs=[(130, 900), (129, 129), (131, 400)], heads=4, kv=2, dim=128, page=64, ty=rlh.F16, window=129),
    "longer": dict(seqs=[(130, 900), (20, 300)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16, window=200),
    "shared": dict(seqs=[(70, 512 + 90), (70, 512 + 70), (5, 700)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=512,
                   window=60, cap=8.0),
    "many": dict(seqs=[(1 + (i * 7) % 40, 40 + (i * 37) % 100) for i in range(270)], heads=4, kv=1, dim=64, page=16,
                 ty=rlh.BF16, window=7),
}


def last_seen(see, first, window):
    """[row, position]: the last `window` of what comes before the batch and the mask's rows."""
    rows = see.shape[0]
    out = np.zeros((rows, first + rows), bool)
    for i in range(rows):
        line = np.concatenate([np.arange(first), first + np.flatnonzero(see[i])])
        out[i, line[-window:]] = True
    return out


@pytest.mark.parametrize("fill", [None, float("nan")])
@pytest.mark.parametrize("name", list(WINDOWED))
def test_a_chain_under_a_window_is_the_attention(name, fill):
    """Tree attention of chains, some longer than the window, and the attention
    of the same rows: both are the 64-bit form that sees the last positions of
    the window; what lies before them may be NaN."""
    case = dict(WINDOWED[name])
    heads, window, cap, shared = case["heads"], case.pop("window"), case.get("cap", 0.0), case.get("shared", 0)
    b, q, out, lse, masks, _ = tree_case(seed=len(name), **case)
    masks.fill_(-1)
    words = masks.shape[1]
    for s, (rows, n) in enumerate(case["seqs"]):
        r0 = int(b.starts[s])
        masks[r0:r0 + rows] = torch.tensor(cref.pack(np.tril(np.ones((rows, rows), bool)), words), device="cuda")
        if fill is not None:  # what no row of the sequence sees
            for j in range(shared, max(shared, n - rows - window + 1)):
                b.k[b.page_of(s, j), :, j % b.page] = fill
                b.v[b.page_of(s, j), :, j % b.page] = fill
    sees = [cref.causal_sees(rows, n, window) for rows, n in case["seqs"]]
    run_tree(b, q, out, heads, masks, lse, cap=cap, window=rlh.WINDOW_DRAFTS | window)
    check_tree(b, q, out, lse, heads, sees, cap=cap)
    other, lse2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    args = rlh.AttnArgs(heads, window, at(q), at(other), q.stride(0), other.stride(0), b.dim ** -0.5, cap, None, None,
                        at(b.shared_table) if shared else None, shared)
    ws = torch.empty(max(16, rlh.paged_attn_workspace(b.kv(), b.desc(), args)), dtype=torch.uint8, device="cuda")
    rlh.paged_attn_lse(b.kv(), b.desc(), args, at(lse2), at(ws), ws.numel(), None, stream())
    check_tree(b, q, other, lse2, heads, sees, cap=cap)


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("name", list(WINDOWED))
def test_trees_under_a_window_that_bounds_them(name, kind):
    """Of the rows of any mask the last `window`; without the flag, or with no
    window beside it, as before."""
    case = dict(WINDOWED[name])
    heads, window, cap = case["heads"], case.pop("window"), case.get("cap", 0.0)
    b, q, out, lse, masks, sees = tree_case(seed=len(name) + 1, kind=kind, **case)
    tight = [last_seen(see[:, n - rows:], n - rows, window) for see, (rows, n) in zip(sees, case["seqs"])]
    loose = [cref.tree_sees(see[:, n - rows:], n - rows, window) for see, (rows, n) in zip(sees, case["seqs"])]
    for w, seen in ((rlh.WINDOW_DRAFTS | window, tight), (window, loose), (rlh.WINDOW_DRAFTS, sees), (0xffffffff, sees)):
        run_tree(b, q, out, heads, masks, lse, cap=cap, window=w)
        check_tree(b, q, out, lse, heads, seen, cap=cap)


def test_a_bounding_window_captured_and_replayed():
    """The masks that the window leaves are made anew by every replay: masks
    and lengths change in between, and eager calls of another window use the
    same workspace."""
    case = dict(WINDOWED["deep"])
    heads, window = case["heads"], case.pop("window")
    b, q, out, lse, masks, sees = tree_case(seed=3, **case)
    ws = run_tree(b, q, out, heads, masks, lse, window=rlh.WINDOW_DRAFTS | window)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        run_tree(b, q, out, heads, masks, lse, window=rlh.WINDOW_DRAFTS | window, ws=ws, st=side.cuda_stream)
    for seed in (3, 4, 5):
        masks.copy_(tree_case(seed=seed, **case)[4])
        sees = tree_case(seed=seed, **case)[5]
        tight = [last_seen(see[:, n - rows:], n - rows, window) for see, (rows, n) in zip(sees, case["seqs"])]
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_tree(b, q, out, lse, heads, tight)
        tighter = [last_seen(see[:, n - rows:], n - rows, 2) for see, (rows, n) in zip(sees, case["seqs"])]
        run_tree(b, q, out, heads, masks, lse, window=rlh.WINDOW_DRAFTS | 2, ws=ws)
        check_tree(b, q, out, lse, heads, tighter)


# ---- empty sequences ------------------------------------------------------------------

def test_a_batch_of_empty_sequences():
    """With max_kv 0 every count is 0 and nothing moves; a sequence that is not empty is skipped."""
    b = ref.Batch([(0, 0), (0, 0), (0, 0)], 2, 64, 16, rlh.F16, seed=1, pad_rows=1)
    b.kv_len[1] = 5
    keep = torch.full((3, 2, 4), 99, dtype=torch.int32, device="cuda")
    count, mass, st = torch.full((3,), 99, dtype=torch.int32, device="cuda"), torch.rand(b.k.shape[:3], device="cuda"), word()
    for stride in (0, b.table.shape[1]):
        seqs = rlh.Seqs(3, 0, 0, 0, stride, None, at(b.kv_len), at(b.table))
        st.zero_()
        rlh.evict_select(b.kv(), seqs, rlh.EvictArgs(at(mass), 4, 1, 1, 4, at(keep), at(count)), at(st), stream())
        assert int(st) == rlh.SERVE_BAD_SEQ and count.tolist() == [0, 0, 0] and torch.all(keep == 99)
        k, m = b.k.clone(), mass.clone()
        st.zero_()
        rlh.paged_move(b.kv(), seqs, rlh.MoveArgs(at(keep), 4, 1, at(count), 4, None, at(mass), at(mass)), at(st), stream())
        assert int(st) == 0 and torch.equal(b.k, k) and torch.equal(mass, m)
