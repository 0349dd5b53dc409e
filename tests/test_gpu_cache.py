"""The operators that edit a paged cache (include/rlh_cache.h) on the GPU
against their plain 64-bit forms (tests/cache_ref.py)."""
import math

import numpy as np
import pytest
import torch

import cache_ref as cref
import rlh
import serve_ref as ref

pytestmark = pytest.mark.gpu

TORCH = ref.TORCH


def stream():
    return torch.cuda.current_stream().cuda_stream


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def ints(x):
    return torch.tensor(np.asarray(x, np.int64).astype(np.uint32).view(np.int32), dtype=torch.int32, device="cuda")


def at(x):
    return None if x is None else x.data_ptr()


# ---- trees: masks and positions ---------------------------------------------------

TREES = {
    "one": [1], "two": [2], "63": [63], "64": [64], "65": [65], "129": [129],
    "ragged": [7, 0, 64, 1, 26, 65, 128, 0, 3], "long": [700, 5, 1000],
}


def tree_batch(sizes, seed, first=None, roots=0.15, reach=9):
    """q_start, kv_len and the parents of a batch of trees, as lists."""
    r = cref.rng(seed)
    trees = [cref.random_tree(r, n, reach, roots) for n in sizes]
    starts = np.cumsum([0] + list(sizes))
    firsts = [r.randrange(0, 500) if first is None else first for _ in sizes]
    return trees, starts, [f + n for f, n in zip(firsts, sizes)]


@pytest.mark.parametrize("with_base", [False, True])
@pytest.mark.parametrize("name", list(TREES))
def test_tree_masks(name, with_base):
    sizes = TREES[name]
    trees, starts, length = tree_batch(sizes, len(name), reach=9 if name != "long" else 3)
    pad, words = 3, (max(sizes) + 63) // 64 + 1
    rows = int(starts[-1]) + pad
    parents = ints([p for t in trees for p in t] + [0] * pad)
    base = [1000 + 17 * s for s in range(len(sizes))]
    masks = torch.full((rows, words), -2, dtype=torch.int64, device="cuda")
    pos = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    q_start, kv_len, b = ints(starts), ints(length), ints(base)
    seqs = rlh.Seqs(len(sizes), rows, max(sizes), max(length), 0, at(q_start), at(kv_len), None)
    st = word()
    rlh.tree_masks(seqs, at(parents), at(b) if with_base else None, at(masks), words, at(pos), at(st), stream())
    want = torch.full_like(masks, -2)
    want_pos = torch.full_like(pos, 77)
    for s, tree in enumerate(trees):
        if not tree:
            continue
        see = cref.mask_matrix(tree)
        a = int(starts[s])
        want[a:a + len(tree)] = torch.tensor(cref.pack(see, words), device="cuda")
        from_ = base[s] if with_base else length[s] - len(tree)
        want_pos[a:a + len(tree)] = torch.tensor(from_ + see.sum(1) - 1, dtype=torch.int32, device="cuda")
    assert int(st) == 0
    assert torch.equal(masks, want) and torch.equal(pos, want_pos)
    # without positions
    masks.fill_(-2)
    rlh.tree_masks(seqs, at(parents), None, at(masks), words, None, None, stream())
    assert torch.equal(masks, want)


def test_tree_masks_of_a_chain_and_of_a_star():
    n = 300
    for tree in ([rlh.NO_PARENT] + list(range(n - 1)), [rlh.NO_PARENT] + [0] * (n - 1), [rlh.NO_PARENT] * n):
        masks = torch.zeros((n, 5), dtype=torch.int64, device="cuda")
        parents, q_start, kv_len = ints(tree), ints([0, n]), ints([n])
        seqs = rlh.Seqs(1, n, n, n, 0, at(q_start), at(kv_len), None)
        rlh.tree_masks(seqs, at(parents), None, at(masks), 5, None, None, stream())
        assert np.array_equal(masks.cpu().numpy(), cref.pack(cref.mask_matrix(tree), 5))


def test_tree_masks_of_parents_that_are_none():
    """A parent at or behind its row is no parent; contradicting sequences are
    left alone."""
    trees = [[rlh.NO_PARENT, 0, 2, 1, 9, 3, 0x80000000, 6], [rlh.NO_PARENT, 0], [0, 0, 1]]
    parents, q_start, kv_len = ints(sum(trees, [])), ints([0, 8, 10, 13]), ints([8, 1, 30])
    masks = torch.full((13, 1), -2, dtype=torch.int64, device="cuda")
    st = word()
    seqs = rlh.Seqs(3, 13, 8, 64, 0, at(q_start), at(kv_len), None)
    rlh.tree_masks(seqs, at(parents), None, at(masks), 1, None, at(st), stream())
    assert int(st) == rlh.SERVE_BAD_SEQ
    got = masks.cpu().numpy()
    assert np.array_equal(got[:8], cref.pack(cref.mask_matrix(trees[0]), 1))
    assert np.all(got[8:10] == -2)
    assert np.array_equal(got[10:], cref.pack(cref.mask_matrix(trees[2]), 1))


# ---- trees: attention ---------------------------------------------------------------

TREE = {
    "one row": dict(seqs=[(1, 1)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "one tree": dict(seqs=[(7, 777)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "tree alone": dict(seqs=[(26, 26), (3, 3), (100, 100)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16),
    "ragged": dict(seqs=[(26, 3000), (5, 40), (0, 7), (1, 500), (63, 1000), (4, 65)], heads=8, kv=2, dim=128, page=16,
                   ty=rlh.BF16, pad_seqs=2, pad_rows=3),
    "small trees": dict(seqs=[(4, 1300), (3, 3), (2, 65), (4, 4), (1, 129), (4, 515)], heads=8, kv=2, dim=128, page=16,
                        ty=rlh.F16),
    "small short": dict(seqs=[(4, 250), (3, 511), (1, 1)], heads=8, kv=2, dim=64, page=32, ty=rlh.BF16),
    "28 over 4": dict(seqs=[(33, 900), (2, 70)], heads=28, kv=4, dim=128, page=64, ty=rlh.BF16),
    "12 over 1": dict(seqs=[(17, 900), (1, 70), (65, 333)], heads=12, kv=1, dim=64, page=128, ty=rlh.F16),
    "24 over 1": dict(seqs=[(9, 300), (2, 31)], heads=24, kv=1, dim=128, page=16, ty=rlh.BF16),
    "64 over 8": dict(seqs=[(63, 5000)], heads=64, kv=8, dim=128, page=64, ty=rlh.F16),
    "wide": dict(seqs=[(300, 700), (150, 160)], heads=4, kv=2, dim=128, page=16, ty=rlh.BF16),
    "cap": dict(seqs=[(20, 300), (4, 900)], heads=8, kv=4, dim=128, page=16, ty=rlh.BF16, cap=5.0, q_scale=6.0),
    "large cap": dict(seqs=[(20, 300), (4, 900)], heads=8, kv=4, dim=64, page=16, ty=rlh.F16, cap=1000.0),
    "window": dict(seqs=[(40, 1000), (3, 900), (1, 5), (30, 64)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, window=64),
    "window in the tree": dict(seqs=[(40, 500), (4, 300), (50, 51)], heads=4, kv=2, dim=128, page=16, ty=rlh.F16, window=3),
    "window 1": dict(seqs=[(33, 100), (2, 900)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16, window=1),
    "shared": dict(seqs=[(9, 512 + 13 * i + 9) for i in range(12)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, shared=512),
    "shared small": dict(seqs=[(3, 300), (1, 257), (30, 400), (2, 258)], heads=16, kv=2, dim=128, page=32, ty=rlh.F16,
                         shared=256),
    "shared window": dict(seqs=[(20, 700), (2, 530), (9, 521)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=512,
                          window=100, cap=8.0, q_scale=3.0),
    "many": dict(seqs=[(1 + (i * 7) % 5, 5 + (i * 37) % 300) for i in range(300)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16),
    "many wide": dict(seqs=[(1 + (i * 7) % 40, 40 + (i * 37) % 100) for i in range(270)], heads=4, kv=1, dim=64, page=16,
                      ty=rlh.BF16),
}


def tree_case(seqs, heads, kv, dim, page, ty, seed=0, cap=0.0, window=0, shared=0, q_scale=1.3, fill=None, pad_seqs=0,
              pad_rows=0, kind="tree"):
    """Masks are a tree's, or any bits (some rows without any)."""
    b = ref.Batch(seqs, kv, dim, page, ty, seed=seed, shared=shared, fill=fill, pad_seqs=pad_seqs, pad_rows=pad_rows)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.zeros((b.n_rows, heads * dim + 8), dtype=TORCH[ty], device="cuda")
    q[:, :heads * dim] = (q_scale * torch.randn((b.n_rows, heads * dim), generator=g)).to(TORCH[ty]).cuda()
    out = torch.full((b.n_rows, heads * dim + 16), 7.0, dtype=TORCH[ty], device="cuda")
    lse = torch.full((b.n_rows, heads), 7.0, device="cuda")
    r, words = cref.rng(seed + 2), (b.max_q + 63) // 64
    bits, sees = np.full((b.n_rows, words), -1, np.int64), []
    for s, (rows, n) in enumerate(seqs):
        if kind == "tree":
            see = cref.mask_matrix(cref.random_tree(r, rows)) if rows else np.zeros((0, 0), bool)
        else:
            see = np.array([[r.random() < (0.0 if i % 5 == 2 else 0.4) for _ in range(rows)] for i in range(rows)], bool)
            see = see.reshape(rows, rows)
        packed = cref.pack(see, words) if rows else np.zeros((0, words), np.int64)
        if kind != "tree" and rows % 64 and rows:
            packed[:, (rows - 1) // 64] |= np.int64(-1) << np.int64(rows % 64)  # bits of no row
        bits[b.starts[s]:b.starts[s] + rows] = packed
        sees.append(cref.tree_sees(see, n - rows, window))
    return b, q, out, lse, torch.tensor(bits, device="cuda"), sees


def run_tree(b, q, out, heads, masks, lse=None, scale=None, cap=0.0, window=0, status=None, ws=None, st=None):
    args = rlh.AttnArgs(heads, window, at(q), at(out), q.stride(0), out.stride(0), b.dim ** -0.5 if scale is None else scale,
                        cap, None, None, at(b.shared_table) if b.shared else None, b.shared)
    if ws is None:
        ws = torch.full((rlh.tree_attn_workspace(b.kv(), b.desc(), args) + 16,), 0xff, dtype=torch.uint8, device="cuda")
    rlh.tree_attn(b.kv(), b.desc(), args, at(masks), masks.shape[1], at(lse), at(ws), ws.numel() // 16 * 16, at(status),
                  stream() if st is None else st)
    return ws


def check_tree(b, q, out, lse, heads, sees, scale=None, cap=0.0):
    want, bound, want_lse, far = cref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, sees,
                                                b.dim ** -0.5 if scale is None else scale, cap)
    n = b.n_live
    got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
    assert not torch.any(torch.isnan(got[:n]))
    assert torch.all(((got - want).abs() - bound - 1e-30)[:n] <= 0), float(((got - want).abs() - bound)[:n].max())
    assert torch.all(out[:, heads * b.dim:] == 7.0) and torch.all(out[n:] == 7.0)
    if lse is not None:
        none = want_lse[:n] == -math.inf
        assert torch.all(lse[:n][none] == -math.inf)
        off = (lse.double() - want_lse).abs()[:n][~none] - far[:n][~none]
        assert off.numel() == 0 or torch.all(off <= 0), float(off.max())
        assert torch.all(lse[n:] == 7.0)


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("name", list(TREE))
def test_tree_attention(name, kind):
    case = dict(TREE[name])
    print("tree attention", name, kind, flush=True)
    b, q, out, lse, masks, sees = tree_case(seed=len(name), kind=kind, **case)
    st = word()
    run_tree(b, q, out, case["heads"], masks, lse, cap=case.get("cap", 0.0), window=case.get("window", 0), status=st)
    torch.cuda.synchronize()
    assert int(st) == 0
    check_tree(b, q, out, lse, case["heads"], sees, cap=case.get("cap", 0.0))


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["ragged", "small trees", "window", "shared small", "wide", "many"])
def test_tree_attention_ignores_what_no_row_may_see(name, fill):
    case = dict(TREE[name])
    b, q, out, lse, masks, sees = tree_case(seed=4, fill=fill, **case)
    run_tree(b, q, out, case["heads"], masks, lse, window=case.get("window", 0))
    torch.cuda.synchronize()
    check_tree(b, q, out, lse, case["heads"], sees)


@pytest.mark.parametrize("name", ["ragged", "small trees", "28 over 4", "wide"])
def test_tree_attention_values_that_only_some_rows_see(name):
    """K and V of a drafted row that are NaN or infinite reach its descendants
    alone."""
    case = dict(TREE[name])
    heads = case["heads"]
    b, q, out, lse, masks, sees = tree_case(seed=6, **case)
    rows, n = case["seqs"][0]
    j = n - rows + rows // 2
    page, slot = b.page_of(0, j), j % b.page
    keep = b.k[page, :, slot].clone(), b.v[page, :, slot].clone()
    want, bound, _, _ = cref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, sees, b.dim ** -0.5)
    mine = torch.zeros(b.n_live, dtype=torch.bool, device="cuda")
    mine[:rows] = torch.tensor(sees[0][:, j], device="cuda")
    assert 0 < int(mine.sum()) < b.n_live
    for pool, bad in ((b.v, math.nan), (b.v, math.inf), (b.k, math.nan)):
        b.k[page, :, slot], b.v[page, :, slot] = keep
        pool[page, :, slot] = bad
        run_tree(b, q, out, heads, masks, lse)
        got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)[:b.n_live]
        hit = got[mine]
        assert torch.all(hit == bad if bad == math.inf else torch.isnan(hit))
        assert torch.all((got - want[:b.n_live]).abs()[~mine] <= bound[:b.n_live][~mine] + 1e-30)


def test_tree_attention_of_a_chain_is_the_attention():
    """A chain sees what comes before it. The two entries divide the positions
    differently, so their f32 sums run in other orders: each is within its bound
    of the 64-bit form, and so the two are within twice that of each other."""
    seqs = [(5, 300), (40, 1000), (1, 7)]
    b, q, out, lse, _, _ = tree_case(seqs, 8, 2, 128, 16, rlh.BF16, seed=9)
    masks = torch.tensor(np.concatenate([cref.pack(np.tril(np.ones((n, n), bool)), 1) for n, _ in seqs]), device="cuda")
    run_tree(b, q, out, 8, masks, lse)
    other, lse2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    args = rlh.AttnArgs(8, 0, at(q), at(other), q.stride(0), other.stride(0), 128 ** -0.5, 0.0, None, None, None, 0)
    ws = torch.empty(max(16, rlh.paged_attn_workspace(b.kv(), b.desc(), args)), dtype=torch.uint8, device="cuda")
    rlh.paged_attn_lse(b.kv(), b.desc(), args, at(lse2), at(ws), ws.numel(), None, stream())
    sees = [cref.causal_sees(r, n) for r, n in seqs]
    for o, ls in ((out, lse), (other, lse2)):
        check_tree(b, q, o, ls, 8, sees)


def test_tree_attention_skips_contradictions_and_missing_pages():
    case = dict(TREE["shared small"])
    heads = case["heads"]
    b, q, out, lse, masks, sees = tree_case(seed=3, **case)
    b.kv_len[1] = 256  # its new row would lie in the shared positions
    st = word()
    run_tree(b, q, out, heads, masks, lse, status=st)
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.all(out[3] == 7.0) and torch.all(lse[3] == 7.0)
    b.kv_len[1] = 257
    out[3, :heads * b.dim], lse[3] = 0, 0
    gone = b.page_of(2, 300)
    b.table[2, 300 // b.page] = b.n_pages
    st.zero_()
    run_tree(b, q, out, heads, masks, lse, status=st)
    assert int(st) == rlh.SERVE_BAD_PAGE
    for j in range(400):
        if b.page_of(2, j) == gone:
            sees[2][:, j] = False
    check_tree(b, q, out, lse, heads, sees)


@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_tree_attention_scales(scale):
    case = dict(TREE["ragged"])
    b, q, out, lse, masks, sees = tree_case(seed=11, **case)
    run_tree(b, q, out, case["heads"], masks, lse, scale=scale)
    check_tree(b, q, out, lse, case["heads"], sees, scale=scale)


# ---- the log of the sums --------------------------------------------------------------

LSE = {
    "decode": dict(seqs=[(1, 5000), (1, 3), (0, 100), (1, 64), (1, 513)], heads=28, kv=4, dim=128, page=64, ty=rlh.BF16),
    "whole": dict(seqs=[(1, 200), (1, 300)], heads=8, kv=2, dim=64, page=16, ty=rlh.F16),
    "prompts": dict(seqs=[(129, 129), (64, 200), (1, 400)], heads=10, kv=2, dim=128, page=32, ty=rlh.F16, pad_rows=2),
    "everything": dict(seqs=[(150, 400), (1, 600), (9, 9)], heads=6, kv=2, dim=64, page=16, ty=rlh.BF16, window=70,
                       bias=True, cap=8.0, prefix=[20, 100, 9]),
    "shared": dict(seqs=[(1, 512 + i * 13 + 1) for i in range(9)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=512),
}


def plain_case(seqs, heads, kv, dim, page, ty, seed=0, cap=0.0, bias=False, window=0, prefix=None, shared=0, pad_rows=0,
               fill=None):
    b = ref.Batch(seqs, kv, dim, page, ty, seed=seed, shared=shared, pad_rows=pad_rows, fill=fill)
    g = torch.Generator().manual_seed(seed + 1)
    q = (1.3 * torch.randn((b.n_rows, heads * dim), generator=g)).to(TORCH[ty]).cuda()
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda") if bias else None
    pre = ints(prefix) if prefix is not None else None
    sees = [cref.causal_sees(r, n, window, prefix[s] if prefix is not None else 0) for s, (r, n) in enumerate(seqs)]
    out = torch.full_like(q, 7.0)
    args = rlh.AttnArgs(heads, window, at(q), at(out), q.stride(0), out.stride(0), dim ** -0.5, cap, at(slopes), at(pre),
                        at(b.shared_table) if shared else None, shared)
    args.hold = (q, out, slopes, pre)
    return b, q.view(-1, heads, dim), out.view(-1, heads, dim), args, slopes, sees


@pytest.mark.parametrize("name", list(LSE))
def test_attention_with_the_log_of_its_sums(name):
    case = dict(LSE[name])
    heads = case["heads"]
    b, q, out, args, slopes, sees = plain_case(seed=len(name), **case)
    ws = torch.full((rlh.paged_attn_workspace(b.kv(), b.desc(), args) + 16,), 0xff, dtype=torch.uint8, device="cuda")
    lse = torch.full((b.n_rows, heads), 7.0, device="cuda")
    rlh.paged_attn_lse(b.kv(), b.desc(), args, at(lse), at(ws), ws.numel() // 16 * 16, None, stream())
    got = out.clone()
    out.fill_(7.0)
    rlh.paged_attn(b.kv(), b.desc(), args, at(ws), ws.numel() // 16 * 16, None, stream())
    assert torch.equal(got, out)
    _, _, want, far = cref.attention(b, q, heads, sees, b.dim ** -0.5, case.get("cap", 0.0), slopes)
    n = b.n_live
    assert torch.all((lse.double() - want).abs()[:n] <= far[:n]) and torch.all(lse[n:] == 7.0)


# ---- append at positions ----------------------------------------------------------------

@pytest.mark.parametrize("inter", [False, True])
def test_append_at_positions(inter):
    """Rows go to their places and are rotated by the positions given."""
    seqs, heads, kv, dim = [(5, 40), (1, 300), (26, 26)], 4, 2, 128
    b = ref.Batch(seqs, kv, dim, 16, rlh.BF16, seed=1, pad_rows=2)
    g = torch.Generator().manual_seed(2)
    x = (1.7 * torch.randn((b.n_rows, (heads + 2 * kv) * dim), generator=g)).cuda()
    f = torch.tensor(rlh.rope_freqs(64, 1e6)[0]).cuda()
    pos = torch.randint(0, 130000, (b.n_rows,), generator=g).cuda()
    q_out = torch.full((b.n_rows, heads * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    size = x.element_size()
    args = rlh.AppendArgs(rlh.F32, heads, at(x), at(x) + heads * dim * size, at(x) + (heads + kv) * dim * size, x.stride(0),
                          x.stride(0), x.stride(0), None, None, 1e-6, 1.0, at(f), 64, int(inter), at(q_out), q_out.stride(0))
    positions = pos.to(torch.int32)
    st = word()
    rlh.paged_append_at(b.kv(), b.desc(), args, at(positions), at(st), stream())
    assert int(st) == 0
    rows = x.double().view(b.n_rows, heads + 2 * kv, dim)
    want = ref.rotate(rows[:, :heads + kv], pos, f, 1.0, 64, inter)
    # a rounding, and f32 angles' sines and cosines (2^-22) of the pair's sizes
    big = rows.abs().amax(-1, keepdim=True) * 2
    tol = want.abs() * 2.0 ** -8 + big[:, :heads + kv] * 2.0 ** -21
    n = b.n_live
    got = q_out.double().view(b.n_rows, heads, dim)
    assert torch.all((got - want[:, :heads]).abs()[:n] <= tol[:, :heads][:n]) and torch.all(q_out[n:] == 7.0)
    for s, (r, total) in enumerate(seqs):
        for i in range(r):
            p, row = total - r + i, int(b.starts[s]) + i
            page, slot = b.page_of(s, p), p % 16
            assert torch.all((b.k[page, :, slot].double() - want[row, heads:]).abs() <= tol[row, heads:])
            assert torch.equal(b.v[page, :, slot], rows[row, heads + kv:].to(torch.bfloat16))
    # the places themselves: the plain append's bits
    k0, q0 = b.k.clone(), q_out.clone()
    rlh.paged_append(b.kv(), b.desc(), args, None, stream())
    k1, q1 = b.k.clone(), q_out.clone()
    for s, (r, total) in enumerate(seqs):
        positions[int(b.starts[s]):int(b.starts[s]) + r] = torch.arange(total - r, total, device="cuda")
    b.k.copy_(k0)
    q_out.copy_(q0)
    rlh.paged_append_at(b.kv(), b.desc(), args, at(positions), None, stream())
    assert torch.equal(b.k, k1) and torch.equal(q_out, q1)


# ---- the kept branch -----------------------------------------------------------------------

def accept_inputs(trees, seed, hit=0.8, vocab=50):
    r = cref.rng(seed)
    tokens = [[r.randrange(vocab) for _ in t] for t in trees]
    sampled = [[r.randrange(vocab) for _ in t] for t in trees]
    for t, tok, drawn in zip(trees, tokens, sampled):
        for i in range(len(t)):
            kids = [c for c in range(i + 1, len(t)) if t[c] == i]
            if kids and r.random() < hit:
                drawn[i] = tok[r.choice(kids)]
    return tokens, sampled


def run_accept(trees, tokens, sampled, length, extra=2, status=None):
    sizes = [len(t) for t in trees]
    keep = [ints(sum(x, []) or [0]) for x in (trees, tokens, sampled)]
    starts, kv_len = ints(np.cumsum([0] + sizes)), ints(length)
    n, most = len(trees), max(sizes + [1])
    path = torch.full((n, most + extra), 99, dtype=torch.int32, device="cuda")
    count, nxt, new_len = (torch.full((n,), 99, dtype=torch.int32, device="cuda") for _ in range(3))
    seqs = rlh.Seqs(n, sum(sizes), most, max(max(length), most), 0, at(starts), at(kv_len), None)
    args = rlh.AcceptArgs(at(keep[0]), at(keep[1]), at(keep[2]), at(path), path.stride(0), at(count), at(nxt), at(new_len))
    rlh.tree_accept(seqs, args, at(status), stream())
    return path.cpu().numpy(), count.cpu().numpy(), nxt.cpu().numpy(), new_len.cpu().numpy()


@pytest.mark.parametrize("name", list(TREES))
def test_accept(name):
    sizes = TREES[name]
    for seed in range(4):
        trees, _, length = tree_batch(sizes, seed, roots=0.02, reach=4)
        tokens, sampled = accept_inputs(trees, seed, hit=0.95, vocab=5 if seed % 2 else 100000)
        st = word()
        path, count, nxt, new_len = run_accept(trees, tokens, sampled, length, status=st)
        assert int(st) == 0
        for s, tree in enumerate(trees):
            if not tree:
                assert count[s] == 0 and nxt[s] == 99 and new_len[s] == 99 and np.all(path[s] == 99)
                continue
            want = cref.accept(tree, tokens[s], sampled[s])
            assert count[s] == len(want) and list(path[s][:len(want)]) == want and np.all(path[s][len(want):] == 99)
            assert nxt[s] == sampled[s][want[-1]] and new_len[s] == length[s] - len(tree) + len(want)


def test_accept_of_a_whole_chain_and_of_contradictions():
    n = 200
    chain = [rlh.NO_PARENT] + list(range(n - 1))
    tokens, sampled = list(range(n)), list(range(1, n + 1))
    path, count, nxt, new_len = run_accept([chain], [tokens], [sampled], [n + 5])
    assert count[0] == n and list(path[0][:n]) == list(range(n)) and nxt[0] == n and new_len[0] == n + 5
    # parents that are not smaller, and tokens beyond 2^31
    big = 0xfffffff0
    path, count, nxt, _ = run_accept([[rlh.NO_PARENT, 1, 0, 2]], [[0, big, big, 7]], [[big, 3, 7, big]], [4])
    assert list(path[0][:3]) == [0, 2, 3] and count[0] == 3 and np.uint32(nxt[0]) == big
    st = word()
    path, count, nxt, _ = run_accept([[rlh.NO_PARENT, 0], [rlh.NO_PARENT]], [[1, 2], [3]], [[2, 9], [4]], [1, 8], status=st)
    assert int(st) == rlh.SERVE_BAD_SEQ and list(count) == [0, 1] and nxt[0] == 99 and nxt[1] == 4


def test_accept_without_rows():
    q_start, kv_len, out = ints([0, 0, 0]), ints([5, 6]), torch.full((6,), 99, dtype=torch.int32, device="cuda")
    seqs = rlh.Seqs(2, 0, 0, 0, 0, at(q_start), at(kv_len), None)
    rlh.tree_accept(seqs, rlh.AcceptArgs(None, None, None, None, 0, at(out), at(out) + 8, at(out) + 16), None, stream())
    assert out.tolist() == [0, 0, 99, 99, 99, 99]


# ---- moving rows ------------------------------------------------------------------------------

def run_move(b, index, count, base=None, mass=None, mass_out=None, per_head=True, status=None, max_count=None):
    """index: [sequence, KV head or 1, j] of whole numbers."""
    idx = ints(index)
    c = ints(count)
    bs = None if base is None else ints(base)
    args = rlh.MoveArgs(at(idx), idx.shape[2], int(per_head), at(c), idx.shape[2] if max_count is None else max_count, at(bs),
                        at(mass), at(mass_out))
    seqs = b.desc()
    seqs.q_start, seqs.n_rows, seqs.max_q = None, 0, 0
    rlh.paged_move(b.kv(), seqs, args, at(status), stream())


def moved(b, index, count, base, arrays, per_head, skip=()):
    """The arrays [page, head, slot, ...] after the move, from copies."""
    old = [x.clone() for x in arrays]
    new = [x.clone() for x in arrays]
    for s in range(len(b.seqs)):
        for g in range(b.kv_heads):
            j = [i for i in range(count[s]) if (s, i) not in skip]
            if not j:
                continue
            src = [int(index[s][g if per_head else 0][i]) + base[s] for i in j]
            dst = [i + base[s] for i in j]
            ps, pd = ([b.page_of(s, x) for x in y] for y in (src, dst))
            ss, sd = ([x % b.page for x in y] for y in (src, dst))
            for o, w in zip(old, new):
                w[pd, g, sd] = o[ps, g, ss]
    return new


MOVES = {
    "one": dict(lengths=[1], count=[1], kv=1, dim=64, page=16),
    "branches": dict(lengths=[100, 40, 777, 16], count=[5, 1, 0, 3], base=[90, 39, 700, 0], kv=3, dim=128, page=16, per_head=False),
    "eviction": dict(lengths=[1000, 333, 2100], count=[400, 333, 77], kv=2, dim=128, page=32),
    "long": dict(lengths=[9000], count=[7000], kv=2, dim=64, page=128),
    "ragged": dict(lengths=[5, 0, 64, 65, 300, 1], count=[3, 0, 64, 10, 299, 1], kv=4, dim=128, page=64),
}


@pytest.mark.parametrize("mass", [None, "in place", "apart"])
@pytest.mark.parametrize("order", ["rising", "any"])
@pytest.mark.parametrize("name", list(MOVES))
def test_move(name, order, mass):
    case = dict(MOVES[name])
    lengths, count, per_head = case["lengths"], case["count"], case.get("per_head", True)
    base = case.get("base")
    r = np.random.default_rng(len(name))
    b = ref.Batch([(0, n) for n in lengths], case["kv"], case["dim"], case["page"], rlh.BF16, seed=2, pad_rows=1)
    lists = case["kv"] if per_head else 1
    index = np.full((len(lengths), lists, max(count) + 3), 0x7fffffff, np.int64)
    for s, n in enumerate(lengths):
        room = n - (base[s] if base else 0)
        for g in range(lists):
            if order == "rising":
                index[s, g, :count[s]] = np.sort(r.choice(room, count[s], replace=False))
            else:  # any place from its own on, some twice
                index[s, g, :count[s]] = [r.integers(j, room) for j in range(count[s])]
    m = torch.rand(b.k.shape[:3], device="cuda")
    out = m if mass == "in place" else torch.zeros_like(m)
    k, v, w = moved(b, index, count, base or [0] * len(lengths), [b.k, b.v, m], per_head)
    if mass == "apart":
        kept = moved(b, index, count, base or [0] * len(lengths), [torch.ones_like(m)], per_head)[0]
        touched = torch.zeros_like(m)
        for s in range(len(lengths)):
            for j in range(count[s]):
                p = j + (base[s] if base else 0)
                touched[b.page_of(s, p), :, p % b.page] = kept[b.page_of(s, p), :, p % b.page]
        w = torch.where(touched > 0, w, 0.0)
    st = word()
    run_move(b, index, count, base, m if mass else None, out if mass else None, per_head, st, max_count=max(count))
    assert int(st) == 0
    assert torch.equal(b.k, k) and torch.equal(b.v, v)
    if mass:
        assert torch.equal(out, w)


def test_move_leaves_out_what_it_cannot():
    """Entries below their place or behind the length, counts past their
    bounds, pages that do not exist: the others go through."""
    lengths = [100, 100, 100, 60]
    b = ref.Batch([(0, n) for n in lengths], 2, 128, 16, rlh.F16, seed=3, pad_rows=1)
    index = np.tile(np.arange(30) * 2, (4, 1, 1))
    index[0, 0, 7] = 3           # below its place
    index[0, 0, 9] = 95          # behind the length from its base on
    index[0, 0, 11] = 0xffffffff
    count, base = [30, 31, 30, 30], [10, 0, 0, 40]
    skip = {(0, 7), (0, 9), (0, 11)} | {(1, j) for j in range(31)} | {(3, j) for j in range(30)}
    wide = np.zeros((4, 1, 31), np.int64)
    wide[:, :, :30] = index
    k, v = moved(b, wide, count, base, [b.k, b.v], False, skip)
    st = word()
    run_move(b, wide, count, base, per_head=False, status=st, max_count=30)
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.equal(b.k, k) and torch.equal(b.v, v)
    # a page that is not there: rows from it stay where they were
    gone = 32 // 16
    b.table[2, gone] = b.n_pages + 5
    count = [0, 0, 30, 0]
    skip = {(2, j) for j in range(30) if (2 * j) // 16 == gone or j // 16 == gone}
    k, v = moved(b, wide, count, [0] * 4, [b.k, b.v], False, skip)
    st.zero_()
    run_move(b, wide, count, per_head=False, status=st, max_count=30)
    assert int(st) == rlh.SERVE_BAD_PAGE
    assert torch.equal(b.k, k) and torch.equal(b.v, v)


# ---- gathered weights ----------------------------------------------------------------------------

MASS = {
    "one": dict(seqs=[(1, 1)], heads=2, kv=1, dim=64, page=16, ty=rlh.F16),
    "decode": dict(seqs=[(1, 777), (1, 3), (0, 50), (1, 128), (1, 129), (1, 2000)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "group 8": dict(seqs=[(1, 500), (2, 2)], heads=16, kv=2, dim=128, page=64, ty=rlh.F16),
    "group 24": dict(seqs=[(1, 500), (2, 31)], heads=24, kv=1, dim=128, page=32, ty=rlh.BF16),
    "last rows": dict(seqs=[(32, 1500), (32, 32), (5, 200)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16),
    "prompt": dict(seqs=[(300, 300), (129, 400)], heads=4, kv=2, dim=64, page=128, ty=rlh.F16),
    "window": dict(seqs=[(20, 900), (1, 500), (3, 64)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, window=100),
    "cap": dict(seqs=[(20, 200), (1, 500)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, cap=7.0),
    "everything": dict(seqs=[(150, 400), (1, 600), (9, 9)], heads=6, kv=2, dim=64, page=16, ty=rlh.BF16, window=70, bias=True,
                       cap=80.0, prefix=[20, 100, 9]),
    "shared": dict(seqs=[(1, 64 + 13 * i + 1) for i in range(9)] + [(3, 70)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=64),
    "many": dict(seqs=[(1, 1 + (i * 37) % 300) for i in range(300)], heads=4, kv=2, dim=64, page=16, ty=rlh.BF16),
}


@pytest.mark.parametrize("decay", [0.0, 1.0, 0.75])
@pytest.mark.parametrize("name", list(MASS))
def test_mass(name, decay):
    case = dict(MASS[name])
    heads, cap = case["heads"], case.get("cap", 0.0)
    b, q, out, args, slopes, sees = plain_case(seed=len(name), fill=float("nan") if name == "decode" else None, **case)
    _, _, want, _ = cref.attention(b, q, heads, sees, b.dim ** -0.5, cap, slopes)
    lse = want.float()
    old = torch.rand(b.k.shape[:3], device="cuda")
    for s, (rows, n) in enumerate(b.seqs):  # nothing is read there
        for j in range(n - rows, n) if decay else range(b.shared, n if rows else 0):
            old[b.page_of(s, j), :, j % b.page] = math.nan
    expect, bound = cref.mass(b, q, heads, sees, lse, b.dim ** -0.5, decay, old, cap, slopes, b.shared)
    got = old.clone()
    st = word()
    rlh.paged_mass(b.kv(), b.desc(), args, at(lse), decay, at(got), at(st), stream())
    assert int(st) == 0
    live = torch.isfinite(expect)
    assert torch.equal(torch.isnan(got), ~live)  # behind the lengths, and in pages of nobody: as it was
    far = ((got.double() - expect).abs() - bound)[live]
    assert torch.all(far <= 0), float(far.max())
    again = old.clone()
    rlh.paged_mass(b.kv(), b.desc(), args, at(lse), decay, at(again), None, stream())
    assert torch.equal(again[live], got[live])


def test_mass_of_rows_without_a_sum_and_of_missing_pages():
    b, q, out, args, _, sees = plain_case([(2, 100), (1, 50)], 4, 2, 128, 16, rlh.BF16, seed=5)
    lse = torch.full((b.n_rows, 4), 1.0, device="cuda")
    lse[0] = -math.inf
    sees[0][0] = False
    old = torch.rand(b.k.shape[:3], device="cuda")
    expect, bound = cref.mass(b, q, 4, sees, lse, 128 ** -0.5, 1.0, old)
    gone = b.page_of(1, 20)
    expect[gone], bound[gone] = old[gone].double(), 0
    b.table[1, 1] = 0x7fffffff
    st = word()
    got = old.clone()
    rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 1.0, at(got), at(st), stream())
    assert int(st) == rlh.SERVE_BAD_PAGE
    assert torch.all((got.double() - expect).abs() <= bound)
    b.kv_len[0] = 1  # fewer positions than rows
    st.zero_()
    got = old.clone()
    rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 1.0, at(got), at(st), stream())
    assert int(st) == rlh.SERVE_BAD_SEQ | rlh.SERVE_BAD_PAGE
    for j in range(100):
        assert torch.equal(got[b.page_of(0, j), :, j % 16], old[b.page_of(0, j), :, j % 16])


# ---- what stays ---------------------------------------------------------------------------------------

def gathered(b, s, g, mass):
    return np.array([float(mass[b.page_of(s, j), g, j % b.page]) for j in range(b.seqs[s][1])], np.float32)


def run_evict(b, mass, budget, first, last, status=None, extra=2):
    most = min(budget, b.max_kv)
    keep = torch.full((len(b.seqs), b.kv_heads, most + extra), 0x7f7f7f7f, dtype=torch.int32, device="cuda")
    count = torch.full((len(b.seqs),), 99, dtype=torch.int32, device="cuda")
    seqs = b.desc()
    seqs.q_start, seqs.n_rows, seqs.max_q = None, 0, 0
    rlh.evict_select(b.kv(), seqs, rlh.EvictArgs(at(mass), budget, first, last, most + extra, at(keep), at(count)),
                     at(status), stream())
    return keep.cpu().numpy(), count.cpu().numpy()


def masses(shape, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "spread":
        return torch.exp(3 * torch.randn(shape, generator=g)).cuda()
    if kind == "ties":
        return (torch.randint(0, 4, shape, generator=g).float() / 4).cuda()
    if kind == "equal":
        return torch.full(shape, 0.25).cuda()
    if kind == "near":  # neighbours in the last bits
        return (1.0 + torch.randint(0, 40, shape, generator=g) * 2.0 ** -23).cuda()
    m = torch.randn(shape, generator=g)  # special values among others
    pick = torch.randint(0, 8, shape, generator=g)
    for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0)):
        m[pick == i] = x
    m[pick == 5] = torch.rand(shape, generator=g)[pick == 5] * 1e-40  # below the normal range
    return m.cuda()


EVICT = [
    # lengths, kv, page, budget, first, last
    ([1], 1, 16, 1, 0, 0), ([2], 2, 16, 1, 0, 0), ([2], 2, 16, 1, 1, 0), ([2], 2, 16, 1, 0, 1),
    ([100, 64, 0, 63, 65], 3, 16, 64, 4, 20), ([1023, 1024, 1025, 1026], 1, 32, 1024, 0, 0),
    ([5000, 10, 700], 2, 64, 256, 16, 240), ([5000], 1, 128, 4999, 1, 1), ([300, 200], 2, 256, 1000, 3, 3),
    ([20000, 4100], 1, 16, 4096, 4, 256),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "near", "special"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(case, kind):
    lengths, kv, page, budget, first, last = EVICT[case]
    b = ref.Batch([(0, n) for n in lengths], kv, 64, page, rlh.F16, seed=case, pad_rows=1)
    m = masses(b.k.shape[:3], kind, case)
    st = word()
    keep, count = run_evict(b, m, budget, first, last, st)
    assert int(st) == 0
    host = m.cpu().numpy()
    for s, n in enumerate(lengths):
        assert count[s] == min(n, budget)
        where = np.array([b.page_of(s, j) for j in range(n)], int), np.arange(n) % page
        for g in range(kv):
            want = cref.evict(host[where[0], g, where[1]], budget, first, last)
            assert np.array_equal(keep[s, g, :count[s]], want), (s, g)
            assert np.all(keep[s, g, count[s]:] == 0x7f7f7f7f)


@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_evict_long(kind):
    """A length beyond any that lies in registers."""
    n, budget = 150001, 30000
    b = ref.Batch([(0, n)], 1, 64, 256, rlh.F16, seed=1, pad_rows=1)
    m = masses(b.k.shape[:3], kind, 3)
    keep, count = run_evict(b, m, budget, 5, 1000)
    where = torch.tensor([b.page_of(0, j) for j in range(0, n, 256)], device="cuda")
    row = m[where, 0].reshape(-1)[:n].cpu().numpy()
    middle = np.argsort(-row[5:n - 1000], kind="stable")[:budget - 1005] + 5
    want = np.concatenate([np.arange(5), np.sort(middle), np.arange(n - 1000, n)])
    assert count[0] == budget and np.array_equal(keep[0, 0, :budget], want)


def test_evict_skips_contradictions_and_missing_pages():
    b = ref.Batch([(0, 100), (0, 80), (0, 60)], 2, 64, 16, rlh.F16, seed=1, pad_rows=1)
    m = masses(b.k.shape[:3], "spread", 2)
    b.kv_len[1] = 101  # past max_kv
    b.table[2, 1] = b.n_pages
    st = word()
    keep, count = run_evict(b, m, 30, 2, 2, st)
    assert int(st) == rlh.SERVE_BAD_SEQ | rlh.SERVE_BAD_PAGE
    assert list(count) == [30, 0, 30] and np.all(keep[1] == 0x7f7f7f7f)
    for s in (0, 2):
        for g in range(2):
            row = gathered(b, s, g, m)
            if s == 2:
                row[16:32] = np.nan
            assert np.array_equal(keep[s, g, :30], cref.evict(row, 30, 2, 2))


# ---- the operators together ---------------------------------------------------------------------------

def test_a_step_with_drafts_captured_and_replayed():
    """Masks, append at the nodes' positions, tree attention, a token per node,
    the accepted branch and its move, as one captured step, for batches whose
    lengths, trees and inputs change from replay to replay; eager calls of the
    program's own lie between. The step is followed on the host: the pages hold
    the kept rows, and the next step's attention sees them."""
    heads, kv, dim, page, vocab, sizes = 8, 2, 64, 16, 200, [26, 7, 1, 70]
    r = cref.rng(3)
    lens = [150, 31, 77, 300]  # positions before the drafts
    room = [(0, n + 6 * 80) for n in lens]
    b = ref.Batch(room, kv, dim, page, rlh.F16, seed=5)
    b.starts = np.cumsum([0] + sizes)
    b.n_rows = b.n_live = int(b.starts[-1])
    b.max_q = max(sizes)
    b.q_start = ints(b.starts)
    n, rows, most, words = len(sizes), b.n_rows, max(sizes), 2
    freqs = torch.tensor(rlh.rope_freqs(dim, 1e4)[0]).cuda()
    x = torch.zeros((rows, (heads + 2 * kv) * dim), device="cuda")
    q_rows = torch.zeros((rows, heads * dim), dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q_rows)
    g = torch.Generator().manual_seed(1)
    w_logits = (0.3 * torch.randn((heads * dim, vocab), generator=g)).cuda()
    parents, tokens, sampled, positions = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(4))
    base = ints(lens)
    masks = torch.zeros((rows, words), dtype=torch.int64, device="cuda")
    path = torch.zeros((n, most), dtype=torch.int32, device="cuda")
    count, nxt, new_len = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    options = torch.tensor(np.frombuffer(b"".join(bytes(rlh.RowSampling(0.0, 0, 1.0, 0.0)) for _ in range(rows)), np.uint8).copy()).cuda()
    u, st = torch.zeros(rows, device="cuda"), word()
    attn = rlh.AttnArgs(heads, 0, at(q_rows), at(out), q_rows.stride(0), out.stride(0), dim ** -0.5, 0.0, None, None, None, 0)
    append = rlh.AppendArgs(rlh.F32, heads, at(x), at(x) + heads * dim * 4, at(x) + (heads + kv) * dim * 4, x.stride(0), x.stride(0),
                            x.stride(0), None, None, 1e-6, 1.0, at(freqs), dim, 0, at(q_rows), q_rows.stride(0))
    accept = rlh.AcceptArgs(at(parents), at(tokens), at(sampled), at(path), most, at(count), at(nxt), at(new_len))
    move = rlh.MoveArgs(at(path), most, 0, at(count), most, at(base), None, None)
    ws = torch.empty(rlh.tree_attn_workspace(b.kv(), b.desc(), attn), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(rlh.sample_rows_workspace(rows, vocab), dtype=torch.uint8, device="cuda")

    def step(s):
        rlh.tree_masks(b.desc(), at(parents), at(base), at(masks), words, at(positions), at(st), s)
        rlh.paged_append_at(b.kv(), b.desc(), append, at(positions), at(st), s)
        rlh.tree_attn(b.kv(), b.desc(), attn, at(masks), words, None, at(ws), ws.numel(), at(st), s)
        logits = out.float() @ w_logits
        rlh.sample_rows(rlh.F32, at(logits), rows, vocab, vocab, at(options), at(u), at(sampled), at(ws2), ws2.numel(), s)
        rlh.tree_accept(b.desc(), accept, at(st), s)
        rlh.paged_move(b.kv(), b.desc(), move, at(st), s)
        return logits

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    now, kept_all = list(lens), 0

    def set_inputs(i):
        trees = [cref.random_tree(r, m, 4) for m in sizes]
        x.copy_(1.2 * torch.randn(x.shape, generator=g))
        parents.copy_(ints(sum(trees, [])))
        b.kv_len.copy_(ints([a + m for a, m in zip(now, sizes)]))
        base.copy_(ints(now))
        # half of the steps draft what the model would draw, found by an eager pass over copies
        drafts = [r.randrange(vocab) for _ in range(rows)]
        return trees, drafts

    with torch.cuda.stream(side):
        out.float() @ w_logits  # the product's library is loaded before the capture
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            logits = step(side.cuda_stream)
    torch.cuda.synchronize()
    for i in range(5):
        trees, drafts = set_inputs(i)
        k0, v0 = b.k.clone(), b.v.clone()
        # an eager pass: what each node draws does not depend on the drafted numbers
        tokens.copy_(ints(drafts))
        torch.cuda.synchronize()
        step(stream())
        drawn = sampled.cpu().numpy().copy()
        for s, tree in enumerate(trees):
            for c in range(1, len(tree)):
                if r.random() < 0.7:
                    drafts[int(b.starts[s]) + c] = int(drawn[int(b.starts[s]) + tree[c]])
        b.k.copy_(k0)
        b.v.copy_(v0)
        tokens.copy_(ints(drafts))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(st) == 0
        assert np.array_equal(sampled.cpu().numpy(), drawn)
        assert torch.equal(logits.argmax(1).to(torch.int32), sampled)
        # attention over what the pages held and the rows just appended
        b.seqs = [(m, a + m) for m, a in zip(sizes, now)]
        sees = [cref.tree_sees(cref.mask_matrix(t), a, 0) for t, a in zip(trees, now)]
        full = b.k.clone(), b.v.clone()
        k1, v1 = k0.clone(), v0.clone()  # the pages before the move
        rowsx = x.double().view(rows, heads + 2 * kv, dim)
        place = torch.tensor([now[s] + len(cref.lineage(t, c)) - 1 for s, t in enumerate(trees) for c in range(len(t))])
        turned = ref.rotate(rowsx[:, :heads + kv], place.cuda(), freqs, 1.0, dim, False)
        for s, m in enumerate(sizes):
            kept = cref.accept(trees[s], drafts[int(b.starts[s]):int(b.starts[s + 1])], drawn[int(b.starts[s]):int(b.starts[s + 1])])
            assert int(count[s]) == len(kept) and path[s, :len(kept)].tolist() == kept
            assert int(nxt[s]) == drawn[int(b.starts[s]) + kept[-1]] and int(new_len[s]) == now[s] + len(kept)
            for c in range(m):
                p, row = now[s] + c, int(b.starts[s]) + c
                v1[b.page_of(s, p), :, p % page] = rowsx[row, heads + kv:].half()
                k1[b.page_of(s, p), :, p % page] = turned[row, heads:].half()
            for j, c in enumerate(kept):  # (keys of a rotation: within the append's bound; values: the same bits)
                p, row = now[s] + j, int(b.starts[s]) + c
                want = turned[row, heads:]
                big = rowsx[row, heads:heads + kv].abs().amax() * 2
                assert torch.all((b.k[b.page_of(s, p), :, p % page].double() - want).abs() <= want.abs() * 2.0 ** -11 + big * 2.0 ** -20)
                assert torch.equal(b.v[b.page_of(s, p), :, p % page], rowsx[row, heads + kv:].half())
            kept_all += len(kept) - 1
        # K as the kernel wrote it: the move changed only kept places, so the attention is checked against the rounded own form
        b.k.copy_(k1)
        b.v.copy_(v1)
        eager = torch.full_like(out, 7.0)
        args = rlh.AttnArgs(heads, 0, at(q_rows), at(eager), q_rows.stride(0), out.stride(0), dim ** -0.5, 0.0, None, None, None, 0)
        rlh.tree_attn(b.kv(), b.desc(), args, at(masks), words, None, at(ws), ws.numel(), None, stream())
        want, bound, _, _ = cref.attention(b, q_rows.view(-1, heads, dim), heads, sees, dim ** -0.5)
        assert torch.all((eager.double().view(-1, heads, dim) - want).abs() <= bound + 1e-30)
        b.k.copy_(full[0])
        b.v.copy_(full[1])
        now = [a + int(c) for a, c in zip(now, count.tolist())]
        b.seqs = [(0, a) for a in now]
    assert kept_all > 10


def test_a_bounded_cache_captured_and_replayed():
    """Attention with its sums, the weights that positions gather, and, when
    the cache is full, the choice and the move: step by step as on the host."""
    heads, kv, dim, page, budget = 8, 2, 128, 16, 96
    lens = [60, 95, 80]
    b = ref.Batch([(1, n + 60) for n in lens], kv, dim, page, rlh.BF16, seed=8)
    q = torch.zeros((3, heads * dim), dtype=torch.bfloat16, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros((3, heads), device="cuda")
    mass = torch.full(b.k.shape[:3], 0.25, device="cuda")
    keep = torch.zeros((3, kv, budget), dtype=torch.int32, device="cuda")
    count, st = torch.zeros(3, dtype=torch.int32, device="cuda"), word()
    args = rlh.AttnArgs(heads, 0, at(q), at(out), q.stride(0), out.stride(0), dim ** -0.5, 0.0, None, None, None, 0)
    ws = torch.empty(max(16, rlh.paged_attn_workspace(b.kv(), b.desc(), args)), dtype=torch.uint8, device="cuda")
    choice = rlh.EvictArgs(at(mass), budget, 4, 16, budget, at(keep), at(count))
    move = rlh.MoveArgs(at(keep), budget, 1, at(count), budget, None, at(mass), at(mass))

    def step(s):
        rlh.paged_attn_lse(b.kv(), b.desc(), args, at(lse), at(ws), ws.numel(), at(st), s)
        rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 0.9, at(mass), at(st), s)
        rlh.evict_select(b.kv(), b.desc(), choice, at(st), s)
        rlh.paged_move(b.kv(), b.desc(), move, at(st), s)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    g = torch.Generator().manual_seed(2)
    now = list(lens)
    cut = 0
    for i in range(12):
        now = [n + 1 for n in now]
        b.seqs = [(1, n) for n in now]
        b.kv_len.copy_(ints(now))
        q.copy_(torch.randn(q.shape, generator=g))
        for s, n in enumerate(now):  # the new position's row
            b.k[b.page_of(s, n - 1), :, (n - 1) % page] = torch.randn((kv, dim), generator=g).bfloat16().cuda()
            b.v[b.page_of(s, n - 1), :, (n - 1) % page] = torch.randn((kv, dim), generator=g).bfloat16().cuda()
        k0, v0, m0 = b.k.clone(), b.v.clone(), mass.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(st) == 0
        got = b.k.clone(), b.v.clone(), mass.clone()
        b.k.copy_(k0)
        b.v.copy_(v0)
        sees = [cref.causal_sees(1, n) for n in now]
        want, bound, want_lse, far = cref.attention(b, q.view(3, heads, dim), heads, sees, dim ** -0.5)
        assert torch.all((out.double().view(3, heads, dim) - want).abs() <= bound + 1e-30)
        assert torch.all((lse.double() - want_lse).abs() <= far)
        expect, off = cref.mass(b, q.view(3, heads, dim), heads, sees, lse, dim ** -0.5, 0.9, m0)
        # the masses that the choice saw are those of an eager call
        eager = m0.clone()
        rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 0.9, at(eager), None, stream())
        assert torch.all((eager.double() - expect).abs() <= off)
        host = eager.cpu().numpy()
        k, v, m = k0.clone(), v0.clone(), eager.clone()
        for s, n in enumerate(now):
            pages, slots = np.array([b.page_of(s, j) for j in range(n)]), np.arange(n) % page
            for h in range(kv):
                kept = cref.evict(host[pages, h, slots], budget, 4, 16)
                assert int(count[s]) == len(kept) and keep[s, h, :len(kept)].tolist() == list(kept)
                to, src = (pages[:len(kept)], h, slots[:len(kept)]), (pages[kept], h, slots[kept])
                k[to], v[to], m[to] = k0[src], v0[src], eager[src]
        assert torch.equal(got[0], k) and torch.equal(got[1], v) and torch.equal(got[2], m)
        b.k.copy_(k)
        b.v.copy_(v)
        cut += sum(n > budget for n in now)
        now = [min(n, budget) for n in now]
    assert cut > 5


def test_cache_two_streams_at_once():
    """Tree attention, masses and the choice on two streams, workspaces of their own: the bits of calls alone."""
    jobs = []
    for i, name in enumerate(("ragged", "28 over 4")):
        case = dict(TREE[name])
        b, q, out, lse, masks, _ = tree_case(seed=30 + i, **case)
        ws = run_tree(b, q, out, case["heads"], masks, lse)
        m = masses(b.k.shape[:3], "spread", i)
        args = rlh.AttnArgs(case["heads"], 0, at(q), None, q.stride(0), 0, b.dim ** -0.5, 0.0, None, None, None, 0)
        rlh.paged_mass(b.kv(), b.desc(), args, at(lse), 0.5, at(m), None, stream())
        keep = torch.zeros((b.desc().n_seq, b.kv_heads, 64), dtype=torch.int32, device="cuda")
        count = torch.zeros(b.desc().n_seq, dtype=torch.int32, device="cuda")
        b.kv_len[len(b.seqs):] = 0
        rlh.evict_select(b.kv(), b.desc(), rlh.EvictArgs(at(m), 64, 4, 8, 64, at(keep), at(count)), None, stream())
        jobs.append((b, q, lse, masks, args, case["heads"], ws, out, masses(b.k.shape[:3], "spread", i), m, keep, count,
                     torch.cuda.Stream()))
    torch.cuda.synchronize()
    hold = []
    for _ in range(6):
        for b, q, lse, masks, args, heads, ws, out, m0, m, keep, count, s in jobs:
            o2, l2, m2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0), m0.clone()
            k2, c2 = torch.zeros_like(keep), torch.zeros_like(count)
            torch.cuda.synchronize()
            hold.append((o2, l2, m2, k2, c2, out, lse, m, keep, count))
        for j, (b, q, lse, masks, args, heads, ws, out, m0, m, keep, count, s) in enumerate(jobs):
            o2, l2, m2, k2, c2 = hold[j - 2][:5]
            run_tree(b, q, o2, heads, masks, l2, ws=ws, st=s.cuda_stream)
            rlh.paged_mass(b.kv(), b.desc(), args, at(l2), 0.5, at(m2), None, s.cuda_stream)
            rlh.evict_select(b.kv(), b.desc(), rlh.EvictArgs(at(m2), 64, 4, 8, 64, at(k2), at(c2)), None, s.cuda_stream)
    torch.cuda.synchronize()
    for o2, l2, m2, k2, c2, out, lse, m, keep, count in hold:
        assert torch.equal(o2, out) and torch.equal(l2, lse) and torch.equal(m2, m)
        assert torch.equal(k2, keep) and torch.equal(c2, count)


def test_tree_one_workspace_for_limits():
    """A workspace of a host's limits holds every smaller call, and nothing behind it is written."""
    heads, kv, dim = 16, 2, 64
    limits = rlh.Seqs(300, 4000, 300, 2000, 125, 1 << 40, 1 << 41, 1 << 42)
    pool = rlh.KvPages(rlh.BF16, kv, dim, 16, 1 << 20, 1 << 43, 1 << 44)
    most = rlh.AttnArgs(heads, 0, 1 << 45, 1 << 46, heads * dim, heads * dim, 0.1, 0.0, None, None, 1 << 47, 256)
    size = rlh.tree_attn_workspace(pool, limits, most)
    ws = torch.full((size + 256,), 0xff, dtype=torch.uint8, device="cuda")
    for seqs, shared in (([(300, 2000)], 0), ([(1, 2000)], 0), ([(3, 300 + i) for i in range(280)], 256), ([(1, 9)] * 300, 0),
                         ([(13, 13 + i) for i in range(290)], 0), ([(130, 700)] * 7, 256)):
        b, q, out, lse, masks, sees = tree_case(seqs, heads, kv, dim, 16, rlh.BF16, seed=2, shared=shared)
        args = rlh.AttnArgs(heads, 0, at(q), at(out), q.stride(0), out.stride(0), dim ** -0.5, 0.0, None, None,
                            at(b.shared_table) if shared else None, shared)
        rlh.tree_attn(b.kv(), b.desc(), args, at(masks), masks.shape[1], at(lse), at(ws), size, None, stream())
        torch.cuda.synchronize()
        assert torch.all(ws[size:] == 0xff)
        check_tree(b, q, out, lse, heads, sees)


@pytest.mark.parametrize("ty", [rlh.BF16])
def test_cache_offsets_past_32_bits(ty):
    """Pages whose values lie past 2^32 elements (9 GB of K and of V)."""
    kv, dim, page = 8, 128, 256
    n_pages = (1 << 32) // (kv * dim * page) + 40
    k, v = (torch.zeros((n_pages, kv, page, dim), dtype=TORCH[ty], device="cuda") for _ in range(2))
    pool = rlh.KvPages(ty, kv, dim, page, n_pages, at(k), at(v))
    g = torch.Generator().manual_seed(4)
    ids = [n_pages - 1, n_pages - 3, 2, n_pages - 2]
    b = ref.Batch([(20, 1000)], kv, dim, page, ty, seed=3)
    for i, p in enumerate(ids):
        k[p], v[p] = b.k[b.page_of(0, i * page)], b.v[b.page_of(0, i * page)]
    table, q_start, kv_len = ints([ids]), ints([0, 20]), ints([1000])
    seqs = rlh.Seqs(1, 20, 20, 1000, 4, at(q_start), at(kv_len), at(table))
    heads = 16
    q = torch.randn((20, heads * dim), generator=g).to(TORCH[ty]).cuda()
    see = cref.mask_matrix(cref.random_tree(cref.rng(1), 20))
    masks = torch.tensor(cref.pack(see, 1), device="cuda")
    out, lse, mass = torch.zeros_like(q), torch.zeros((20, heads), device="cuda"), torch.rand((n_pages, kv, page), device="cuda")
    args = rlh.AttnArgs(heads, 0, at(q), at(out), q.stride(0), out.stride(0), dim ** -0.5, 0.0, None, None, None, 0)
    ws = torch.empty(rlh.tree_attn_workspace(pool, seqs, args), dtype=torch.uint8, device="cuda")
    rlh.tree_attn(pool, seqs, args, at(masks), 1, at(lse), at(ws), ws.numel(), None, stream())
    want, bound, want_lse, far = cref.attention(b, q.view(20, heads, dim), heads, [cref.tree_sees(see, 980, 0)], dim ** -0.5)
    assert torch.all((out.double().view(20, heads, dim) - want).abs() <= bound) and torch.all((lse.double() - want_lse).abs() <= far)
    small = torch.zeros(b.k.shape[:3], device="cuda")
    for i, p in enumerate(ids):
        small[b.page_of(0, i * page)] = mass[p]
    for rows in (20, 1):
        qr, ls = q[20 - rows:], lse[20 - rows:].contiguous()
        b.seqs, b.starts = [(rows, 1000)], np.array([0, rows])
        starts = ints([0, rows])
        one = rlh.Seqs(1, rows, rows, 1000, 4, at(starts), at(kv_len), at(table))
        a2 = rlh.AttnArgs(heads, 0, at(qr), None, q.stride(0), 0, dim ** -0.5, 0.0, None, None, None, 0)
        expect, off = cref.mass(b, qr.view(rows, heads, dim), heads, [cref.causal_sees(rows, 1000)], ls, dim ** -0.5, 1.0, small)
        got = mass.clone()
        rlh.paged_mass(pool, one, a2, at(ls), 1.0, at(got), None, stream())
        for i, p in enumerate(ids):
            e = (got[p].double() - expect[b.page_of(0, i * page)]).abs() - off[b.page_of(0, i * page)]
            live = min(page, 1000 - i * page)
            assert torch.all(e[:, :live] <= 0)
    index = ints(np.sort(np.random.default_rng(1).choice(1000, 600, replace=False)))
    c = ints([600])
    rows_k = torch.cat([k[p] for p in ids], 1)[:, :1000][:, index.long()].clone()
    rlh.paged_move(pool, seqs, rlh.MoveArgs(at(index), 600, 0, at(c), 600, None, None, None), None, stream())
    assert torch.equal(torch.cat([k[p] for p in ids], 1)[:, :600], rows_k)


def test_cache_refused_on_the_device():
    """Host memory, and nothing written by a refused call."""
    b, q, out, lse, masks, _ = tree_case([(5, 300)], 4, 2, 64, 16, rlh.F16, seed=1)
    host = torch.zeros(4096, dtype=torch.int64)
    args = rlh.AttnArgs(4, 0, at(q), at(out), q.stride(0), out.stride(0), 0.125, 0.0, None, None, None, 0)
    ws = torch.empty(rlh.tree_attn_workspace(b.kv(), b.desc(), args), dtype=torch.uint8, device="cuda")
    c = word()
    calls = [
        lambda: rlh.tree_attn(b.kv(), b.desc(), args, host.data_ptr(), 1, None, at(ws), ws.numel(), None, stream()),
        lambda: rlh.tree_attn(b.kv(), b.desc(), args, at(masks), 1, host.data_ptr(), at(ws), ws.numel(), None, stream()),
        lambda: rlh.tree_attn(b.kv(), b.desc(), args, at(masks), 1, None, at(ws), 16, None, stream()),
        lambda: rlh.tree_masks(b.desc(), host.data_ptr(), None, at(masks), 1, None, None, stream()),
        lambda: rlh.paged_mass(b.kv(), b.desc(), args, host.data_ptr(), 0.5, at(ws), None, stream()),
        lambda: rlh.paged_move(b.kv(), b.desc(), rlh.MoveArgs(host.data_ptr(), 8, 0, at(c), 8, None, None, None), None, stream()),
        lambda: rlh.evict_select(b.kv(), b.desc(), rlh.EvictArgs(at(ws), 8, 0, 0, 8, host.data_ptr(), at(c)), None, stream()),
    ]
    keep = masks.clone()
    for f in calls:
        with pytest.raises(rlh.RlhError) as e:
            f()
        assert e.value.code == rlh.RLH_EINVAL
    torch.cuda.synchronize()
    assert torch.all(out == 7.0) and torch.all(lse == 7.0) and torch.equal(masks, keep)


@pytest.mark.parametrize("many", [False, True])
def test_tree_attention_with_starts_that_fall(many):
    """A sequence whose start falls is skipped; rows between that two others
    name are written by one of them, and nothing else changes."""
    n = 270 if many else 3
    seqs = [(20, 200), (30, 100), (25, 130)] + [(0, 5)] * (n - 3)
    b, q, out, lse, masks, sees = tree_case(seqs, 8, 2, 64, 16, rlh.F16, seed=13)
    # rows 0 .. 19, then a fall from 50 to 40, then rows 40 .. 74
    starts = b.q_start.clone()
    starts[1], starts[2] = 50, 40
    keep = b.q_start.clone()
    b.q_start.copy_(starts)
    b.max_q = 60
    st = word()
    masks = torch.zeros((b.n_rows, 1), dtype=torch.int64, device="cuda")
    run_tree(b, q, out, 8, masks, lse, status=st)
    torch.cuda.synchronize()
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.all(out[:, 8 * 64:] == 7.0)
    b.q_start.copy_(keep)


def test_tree_attention_of_many_heads():
    """More KV heads than the card has CUs: a block to a head."""
    b, q, out, lse, masks, sees = tree_case([(20, 70), (1, 33)], 300, 300, 64, 16, rlh.BF16, seed=14)
    run_tree(b, q, out, 300, masks, lse)
    check_tree(b, q, out, lse, 300, sees)
