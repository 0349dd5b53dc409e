"""The operators that edit a paged cache (include/rlh_cache.h) where their
kernels go on for long or reach a limit, against the 64-bit forms of
tests/cache_ref.py."""
import numpy as np
import pytest
import torch

import cache_ref as cref
import rlh
import serve_ref as ref
from test_gpu_cache import (at, check_tree, masses, moved, plain_case, run_evict, run_move, run_tree, stream, tree_case,
                            word)

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


def test_the_flag_changes_nothing_where_a_window_bounds_all_rows():
    """One set of arguments serves a layer's entries: attention and weights with
    the flag are those without it."""
    seqs, heads = [(40, 300), (3, 64), (1, 700)], 8
    for window in (0, 5, 100):
        got = []
        for flag in (0, rlh.WINDOW_DRAFTS):
            b, q, out, args, _, sees = plain_case(seqs, heads, 2, 64, 16, rlh.F16, seed=2, window=window)
            args.window |= flag
            lse, mass = torch.full((b.n_rows, heads), 7.0, device="cuda"), torch.ones(b.k.shape[:3], device="cuda")
            ws = torch.empty(max(16, rlh.paged_attn_workspace(b.kv(), b.desc(), args)), dtype=torch.uint8, device="cuda")
            rlh.paged_attn_lse(b.kv(), b.desc(), args, at(lse), at(ws), ws.numel(), None, stream())
            rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 0.5, at(mass), None, stream())
            want, bound, _, _ = cref.attention(b, q, heads, sees, 0.125)
            assert torch.all((out.double() - want).abs() <= bound + 1e-30)
            got.append((out, lse, mass))
        assert all(torch.equal(x, y) for x, y in zip(*got))


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


# ---- jobs of many steps -----------------------------------------------------------------
# Few blocks share the line of a KV head where there are many of them, so that one
# walks past 16 and 32 steps of a tile, whose page ids it holds 16 at a time.
# (tests/test_cache_edges.py finds out how many.)

LONG_JOBS = {
    "pages of 16": dict(seqs=[(20, 10000)], heads=64, kv=64, dim=64, page=16, ty=rlh.BF16),
    "pages of 128": dict(seqs=[(26, 9001), (3, 4000)], heads=128, kv=64, dim=128, page=128, ty=rlh.F16),
    "wide tiles": dict(seqs=[(130, 6000), (3, 700)], heads=128, kv=64, dim=64, page=32, ty=rlh.F16),
    "shared": dict(seqs=[(9, 8192 + 2500), (20, 8192 + 100), (1, 8192 + 1)], heads=64, kv=64, dim=64, page=16, ty=rlh.BF16,
                   shared=8192),
    "shared, capped": dict(seqs=[(40, 9216 + 300), (3, 9216 + 40)], heads=128, kv=64, dim=128, page=64, ty=rlh.F16, shared=9216,
                           cap=6.0),
    "window": dict(seqs=[(20, 9000), (20, 6000)], heads=64, kv=64, dim=64, page=16, ty=rlh.BF16, window=5000),
}


@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("name", list(LONG_JOBS))
def test_tree_attention_of_long_jobs(name, missing):
    """Positions of every third step are far larger in V, so that a step taken
    twice or left out shows; pages are missing in the first, the second and
    the third 16 steps of the line's first job."""
    case = dict(LONG_JOBS[name])
    heads, cap, window, shared = case["heads"], case.get("cap", 0.0), case.pop("window", 0), case.get("shared", 0)
    print("long jobs", name, missing, flush=True)
    b, q, out, lse, masks, sees = tree_case(seed=len(name), window=window, **case)
    for p in range(0, b.n_pages, 3):
        b.v[p] *= 4
    gone = []
    if missing:
        rows, n = case["seqs"][0]
        begin = 0 if shared else max(0, n - rows - window) // 16 * 16 if window else 0
        for step in (2, 17, 18, 31, 35):
            j = begin + 64 * step + 20
            gone.append(b.page_of(0, j))
            if j < shared:
                b.shared_table[j // b.page] = b.n_pages + step
            else:
                b.table[0, j // b.page] = 0x7fffffff - step
        for s, (_, n) in enumerate(case["seqs"]):
            for j in range(n):
                if b.page_of(s, j) in gone:
                    sees[s][:, j] = False
    st = word()
    ws = run_tree(b, q, out, heads, masks, lse, cap=cap, window=window, status=st)
    assert int(st) == (rlh.SERVE_BAD_PAGE if missing else 0)
    check_tree(b, q, out, lse, heads, sees, cap=cap)
    # once more, over what the first call left in the workspace: the same bits
    again, lse2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    run_tree(b, q, again, heads, masks, lse2, cap=cap, window=window, ws=ws)
    assert torch.equal(again, out) and torch.equal(lse2, lse)


# ---- weights, more steps than blocks ------------------------------------------------------
# (which of them go on from step to step: tests/test_cache_edges.py)

GOES_ON = {
    "tokens": dict(seqs=[(1, 1 + (i * 397) % 2600) for i in range(60)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "drafts": dict(seqs=[(4, 4 + (i * 397) % 2000) for i in range(160)], heads=16, kv=4, dim=64, page=64, ty=rlh.F16),
    "tokens, window": dict(seqs=[(1, 1 + (i * 397) % 2600) for i in range(60)], heads=8, kv=8, dim=64, page=32, ty=rlh.F16,
                           window=700, cap=9.0),
    "tokens, shared": dict(seqs=[(2, 258 + (i * 397) % 2600) for i in range(60)], heads=8, kv=8, dim=64, page=32, ty=rlh.BF16,
                           shared=256, bias=True),
    "rows": dict(seqs=[(40, 1500), (20, 700), (1, 900), (150, 333)] + [(0, 5)] * 4096, heads=32, kv=16, dim=128, page=16, ty=rlh.BF16),
    "rows, window": dict(seqs=[(40, 1500), (200, 700), (3, 900)] + [(0, 5)] * 4096, heads=16, kv=16, dim=64, page=64, ty=rlh.F16,
                         window=130, prefix=[300, 20, 1] + [0] * 4096),
    "rows, two blocks": dict(seqs=[(40, 1500), (200, 700), (3, 900)] + [(0, 5)] * 2045, heads=32, kv=16, dim=64, page=16, ty=rlh.F16,
                             cap=80.0),
}


@pytest.mark.parametrize("decay", [0.0, 0.75])
@pytest.mark.parametrize("name", list(GOES_ON))
def test_mass_of_more_steps_than_blocks(name, decay):
    case = dict(GOES_ON[name])
    heads, cap = case["heads"], case.get("cap", 0.0)
    b, q, out, args, slopes, sees = plain_case(seed=len(name), **case)
    live = [s for s, (rows, _) in enumerate(case["seqs"]) if rows]
    sees = [see if s in live else None for s, see in enumerate(sees)]
    _, _, want, _ = cref.attention(b, q, heads, sees, b.dim ** -0.5, cap, slopes)
    lse = want.float()
    old = torch.rand(b.k.shape[:3], device="cuda")
    expect, bound = cref.mass(b, q, heads, sees, lse, b.dim ** -0.5, decay, old, cap, slopes, b.shared)
    # A term below 2^-126 may count as none (the bias puts far positions there): each of a
    # position's terms, rows times heads of a group, is then off by less than 2^-126, and
    # the factor beside the exponential is below 1 + 2^-20.
    bound += max(q for q, _ in case["seqs"]) * (heads // b.kv_heads) * 2.0 ** -126 * (1 + 2.0 ** -20)
    # a page that is not there, in the last steps of the longest sequence
    long = max(live, key=lambda s: case["seqs"][s][1])
    j = (case["seqs"][long][1] - 200) // b.page
    gone = b.page_of(long, j * b.page)
    for missing in (False, True):
        if missing:
            b.table[long, j] = b.n_pages
            expect[gone], bound[gone] = old[gone].double(), 0
        got, st = old.clone(), word()
        rlh.paged_mass(b.kv(), b.desc(), args, at(lse), decay, at(got), at(st), stream())
        assert int(st) == (rlh.SERVE_BAD_PAGE if missing else 0)
        far = (got.double() - expect).abs() - bound
        assert torch.all(far <= 0), float(far.max())


# ---- the choice at the limits of its forms --------------------------------------------------

def kept(row, budget, first, last):
    """cref.evict for long rows."""
    n = len(row)
    if n <= budget:
        return np.arange(n)
    j = np.arange(first, n - last)
    x = row[j]
    order = np.lexsort((j, -np.where(np.isnan(x), 0.0, x), np.isnan(x)))
    return np.concatenate([np.arange(first), np.sort(j[order[:budget - first - last]]), np.arange(n - last, n)])


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("n", [8192, 8193, 16384, 16385, 40960, 40961])
def test_evict_at_the_limits_of_its_forms(n, kind):
    lengths, budget, first, last = [n, n - 1, 700, n - 5000], n // 3, 7, 300
    b = ref.Batch([(0, x) for x in lengths], 2, 64, 64, rlh.F16, seed=n, pad_rows=1)
    m = masses(b.k.shape[:3], kind, n)
    for budget in (n // 3, n - 1):
        st = word()
        keep, count = run_evict(b, m, budget, first, last, st)
        assert int(st) == 0
        host = m.cpu().numpy()
        for s, x in enumerate(lengths):
            where = np.array([b.page_of(s, i) for i in range(x)], int), np.arange(x) % 64
            assert count[s] == min(x, budget)
            for g in range(2):
                assert np.array_equal(keep[s, g, :count[s]], kept(host[where[0], g, where[1]], budget, first, last)), (s, g)
                assert np.all(keep[s, g, count[s]:] == 0x7f7f7f7f)


@pytest.mark.parametrize("order", ["rising", "any"])
@pytest.mark.parametrize("dim", [64, 128])
def test_move_in_many_rounds(dim, order):
    """Lists of several rounds of 2048 rows, with their masses, in place."""
    lengths, count = [9000, 4100, 6500], [7000, 4099, 2049]
    b = ref.Batch([(0, n) for n in lengths], 2, dim, 32, rlh.BF16, seed=dim, pad_rows=1)
    r = np.random.default_rng(dim)
    index = np.zeros((3, 2, max(count)), np.int64)
    for s, n in enumerate(lengths):
        for g in range(2):
            index[s, g, :count[s]] = (np.sort(r.choice(n, count[s], replace=False)) if order == "rising" else
                                      [r.integers(j, min(n, j + 3000)) for j in range(count[s])])
    m = torch.rand(b.k.shape[:3], device="cuda")
    k, v, w = moved(b, index, count, [0] * 3, [b.k, b.v, m], True)
    st = word()
    run_move(b, index, count, mass=m, mass_out=m, status=st)
    assert int(st) == 0
    assert torch.equal(b.k, k) and torch.equal(b.v, v) and torch.equal(m, w)


# ---- starts that fall -----------------------------------------------------------------------

@pytest.mark.parametrize("many", [False, True])
def test_tree_attention_with_starts_that_fall_row_by_row(many):
    """Rows 0 .. 49 are the first sequence's, 40 .. 74 the third's, between
    them one is skipped: rows of one owner are its own, rows of two one of
    theirs, all others as they were."""
    n = 270 if many else 3
    seqs = [(20, 200), (30, 100), (25, 130)] + [(0, 5)] * (n - 3)
    b, q, out, lse, _, _ = tree_case(seqs, 8, 2, 64, 16, rlh.F16, seed=13, pad_rows=4)
    b.q_start[1], b.q_start[2] = 50, 40
    b.max_q = 60
    masks, st = torch.zeros((b.n_rows, 1), dtype=torch.int64, device="cuda"), word()
    run_tree(b, q, out, 8, masks, lse, status=st)
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.all(out[:, 8 * 64:] == 7.0) and torch.all(out[75:] == 7.0) and torch.all(lse[75:] == 7.0)
    got = out[:, :8 * 64].double().view(-1, 8, 64)
    near = []
    for s, r0, rows, n in ((0, 0, 50, 200), (2, 40, 35, 130)):
        b.starts[s], live = r0, list(seqs)
        b.seqs = [(rows, n) if i == s else (0, 5) for i in range(len(live))]
        see = np.zeros((rows, n), bool)
        see[:, :n - rows] = True
        want, bound, want_lse, far = cref.attention(b, q[:, :8 * 64].view(-1, 8, 64), 8, {s: see}, 0.125)
        near.append((((got - want).abs() <= bound + 1e-30).all(-1)) & ((lse.double() - want_lse).abs() <= far))
    assert near[0][:40].all() and near[1][50:75].all() and (near[0] | near[1])[40:50].all()
