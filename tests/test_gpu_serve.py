"""The batched serving operators (include/rlh_serve.h) on the GPU against
their plain 64-bit forms (tests/serve_ref.py)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import rlh
import serve_ref as ref

pytestmark = pytest.mark.gpu

TORCH = ref.TORCH


def half(ty):
    return torch.finfo(TORCH[ty]).eps / 2


def stream():
    return torch.cuda.current_stream().cuda_stream


def status_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ---- append -------------------------------------------------------------------

def append_inputs(b, heads, in_ty, seed, gap=0):
    """q, k and v rows as slices of one buffer with `gap` values behind them."""
    g = torch.Generator().manual_seed(seed)
    width = (heads + 2 * b.kv_heads) * b.dim + gap
    x = (1.7 * torch.randn((b.n_rows, width), generator=g)).to(TORCH[in_ty]).cuda()
    return x


def run_append(b, x, in_ty, heads, q_out, q_norm, k_norm, freqs, mag, rot, inter, status=None, st=None):
    h, g, d = heads, b.kv_heads, b.dim
    at, size = x.data_ptr(), x.element_size()
    args = rlh.AppendArgs(in_ty, h, at, at + h * d * size, at + (h + g) * d * size, x.stride(0), x.stride(0),
                          x.stride(0), None if q_norm is None else q_norm.data_ptr(),
                          None if k_norm is None else k_norm.data_ptr(), 1e-6, mag,
                          None if freqs is None else freqs.data_ptr(), rot, int(inter), q_out.data_ptr(),
                          q_out.stride(0))
    rlh.paged_append(b.kv(), b.desc(), args, None if status is None else status.data_ptr(),
                     stream() if st is None else st)


def append_expected(b, x, heads, q_norm, k_norm, freqs, mag, rot, inter):
    """q, k, v rows in 64 bits and how far the f32 arithmetic may be off
    before the one rounding: a norm of D squares is off by less than
    (D + 8) 2^-24 of the value, the angle's sine and cosine by 2^-22 (2^-23.3
    for the rounded turn, 2^-24 each for sincospi and the magnitude), a
    rotated value by twice that of the pair's sum of magnitudes."""
    d, g = b.dim, b.kv_heads
    xs = x[:, :(heads + 2 * g) * d].double().view(-1, heads + 2 * g, d)
    pos = torch.zeros(b.n_rows, dtype=torch.int64, device="cuda")
    for s, (rows, n) in enumerate(b.seqs):
        r0 = int(b.starts[s])
        pos[r0:r0 + rows] = torch.arange(n - rows, n, device="cuda")
    q = ref.norm(xs[:, :heads], q_norm, float(np.float32(1e-6)))
    k = ref.norm(xs[:, heads:heads + g], k_norm, float(np.float32(1e-6)))
    mags = [q.abs(), k.abs()]
    if rot:
        big = []
        for t in (q, k):
            a = t.abs()
            if inter:
                m = a[..., 0:rot:2] + a[..., 1:rot:2]
                a = torch.cat([m.repeat_interleave(2, -1), a[..., rot:]], -1)
            else:
                m = a[..., :rot // 2] + a[..., rot // 2:rot]
                a = torch.cat([m, m, a[..., rot:]], -1)
            big.append(a * max(1.0, mag))
        mags = big
        q = ref.rotate(q, pos, freqs, mag, rot, inter)
        k = ref.rotate(k, pos, freqs, mag, rot, inter)
    off = (d + 8) * 2.0 ** -24 + 2 * 2.0 ** -22
    return q, k, xs[:, heads + g:], mags[0] * off, mags[1] * off, pos


APPEND = [
    # seqs, heads, kv, dim, page, type, in, rot, inter, norm, gap
    ([(1, 1)], 16, 8, 128, 16, rlh.BF16, rlh.F32, 128, False, True, 0),
    ([(1, 130001)], 4, 2, 128, 256, rlh.F16, rlh.F16, 128, True, False, 8),
    ([(1, 17), (1, 16), (1, 33), (0, 5), (1, 1)], 32, 8, 128, 16, rlh.F16, rlh.BF16, 64, False, True, 4 * 2),
    ([(5, 5), (31, 70), (1, 1000), (130, 130)], 7, 7, 64, 32, rlh.BF16, rlh.F32, 32, True, True, 4),
    ([(700, 911), (3, 3)], 12, 1, 128, 64, rlh.F16, rlh.F32, 16, False, True, 0),
    ([(33, 33)], 6, 2, 64, 16, rlh.BF16, rlh.BF16, 0, False, True, 0),
    ([(9, 20)], 3, 3, 128, 128, rlh.F16, rlh.F16, 0, False, False, 0),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case):
    seqs, heads, kv, dim, page, ty, in_ty, rot, inter, with_norm, gap = APPEND[case]
    b = ref.Batch(seqs, kv, dim, page, ty, seed=case, pad_seqs=case % 3, pad_rows=case % 2 * 3)
    x = append_inputs(b, heads, in_ty, case + 50, gap)
    w = [1 + 0.1 * torch.randn(dim, generator=torch.Generator().manual_seed(9 + i)).cuda() if with_norm else None
         for i in range(2)]
    mag = 1.25 if case % 2 else 1.0
    f = torch.tensor(rlh.rope_freqs(rot, 1e6)[0]).cuda() if rot else None
    q_out = torch.full((b.n_rows, heads * dim + 16), 7.0, dtype=TORCH[ty], device="cuda")
    k0, v0 = b.k.clone(), b.v.clone()
    st = status_word()
    run_append(b, x, in_ty, heads, q_out, w[0], w[1], f, mag, rot, inter, st)
    torch.cuda.synchronize()
    assert int(st) == 0
    q, k, v, q_off, k_off, pos = append_expected(b, x, heads, w[0], w[1], f, mag, rot, inter)
    n, h2 = b.n_live, half(ty)
    got = q_out[:, :heads * dim].double().view(-1, heads, dim)
    assert torch.all((got - q)[:n].abs() <= (q.abs() * h2 + q_off * (1 + h2) + 2.0 ** -25)[:n])
    assert torch.all(q_out[:, heads * dim:] == 7.0) and torch.all(q_out[n:] == 7.0)
    want_k, want_v, seen = k0.double(), v0, torch.zeros(b.k.shape[:1] + b.k.shape[2:3], dtype=torch.bool)
    tol = torch.zeros_like(want_k)
    want_v = v0.clone()
    for s, (rows, total) in enumerate(seqs):
        for i in range(rows):
            p, r = total - rows + i, int(b.starts[s]) + i
            page_id, slot = b.page_of(s, p), p % page
            want_k[page_id, :, slot] = k[r]
            tol[page_id, :, slot] = k[r].abs() * h2 + k_off[r] * (1 + h2) + 2.0 ** -25
            want_v[page_id, :, slot] = v[r].to(TORCH[ty])
    assert torch.all((b.k.double() - want_k).abs() <= tol)  # untouched slots: equal
    assert torch.equal(b.v, want_v)


def test_append_bad_pages_and_sequences():
    """A page id that does not exist takes neither K nor V, sequences whose
    numbers contradict each other are skipped, the others go through."""
    seqs = [(3, 20), (4, 40), (2, 2)]
    b = ref.Batch(seqs, 2, 128, 16, rlh.BF16, seed=3)
    x = append_inputs(b, 4, rlh.F32, 4)
    b.table[0, 1] = b.n_pages  # positions 16..31 of sequence 0: all its new rows
    k0, v0 = b.k.clone(), b.v.clone()
    q_out = torch.full((b.n_rows, 4 * 128), 7.0, dtype=torch.bfloat16, device="cuda")
    st = status_word()
    f = torch.tensor(rlh.rope_freqs(128, 1e4)[0]).cuda()
    run_append(b, x, rlh.F32, 4, q_out, None, None, f, 1.0, 128, False, st)
    assert int(st) == rlh.SERVE_BAD_PAGE
    keep = torch.ones(b.n_pages, dtype=torch.bool)
    for s in (1, 2):
        for p in range(seqs[s][1] - seqs[s][0], seqs[s][1]):
            keep[b.page_of(s, p)] = False
    assert torch.equal(b.k[keep.cuda()], k0[keep.cuda()]) and torch.equal(b.v[keep.cuda()], v0[keep.cuda()])
    assert not torch.any(torch.all(q_out == 7.0, dim=1))
    # a length below the new rows, above max_kv
    for wrong in (2, 41):
        b.kv_len[1] = wrong
        st.zero_()
        q_out.fill_(7.0)
        run_append(b, x, rlh.F32, 4, q_out, None, None, f, 1.0, 128, False, st)
        assert int(st) & rlh.SERVE_BAD_SEQ
        assert torch.all(q_out[3:7] == 7.0) and not torch.any(torch.all(q_out[7:] == 7.0, dim=1))


# ---- attention ------------------------------------------------------------------

def run_attn(b, q, out, heads, scale=None, cap=0.0, slopes=None, window=0, prefix=None, status=None, ws=None, st=None):
    args = rlh.AttnArgs(heads, window, q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0),
                        b.dim ** -0.5 if scale is None else scale, cap, None if slopes is None else slopes.data_ptr(),
                        None if prefix is None else prefix.data_ptr(),
                        b.shared_table.data_ptr() if b.shared else None, b.shared)
    need = rlh.paged_attn_workspace(b.kv(), b.desc(), args)
    if ws is None:
        # what an earlier call may have left there: NaN patterns
        ws = torch.full((need + 16,), 0xff, dtype=torch.uint8, device="cuda")
    rlh.paged_attn(b.kv(), b.desc(), args, ws.data_ptr(), ws.numel() // 16 * 16,
                   None if status is None else status.data_ptr(), stream() if st is None else st)
    return ws


def attn_case(seqs, heads, kv, dim, page, ty, seed=0, cap=0.0, bias=False, window=0, prefix=None, shared=0, q_scale=1.3,
              fill=None, pad_seqs=0, pad_rows=0):
    b = ref.Batch(seqs, kv, dim, page, ty, seed=seed, shared=shared, fill=fill, pad_seqs=pad_seqs, pad_rows=pad_rows)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.zeros((b.n_rows, heads * dim + 8), dtype=TORCH[ty], device="cuda")
    q[:, :heads * dim] = (q_scale * torch.randn((b.n_rows, heads * dim), generator=g)).to(TORCH[ty]).cuda()
    out = torch.full((b.n_rows, heads * dim + 16), 7.0, dtype=TORCH[ty], device="cuda")
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32,
                          device="cuda") if bias else None
    pre = None if prefix is None else torch.tensor(list(prefix) + [0] * pad_seqs, dtype=torch.int32, device="cuda")
    return b, q, out, dict(cap=cap, slopes=slopes, window=window, prefix=pre)


def check_attn(b, q, out, heads, opts, hidden_pages=()):
    want, bound = ref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, b.dim ** -0.5, opts["cap"],
                                opts["slopes"], opts["window"], opts["prefix"], hidden_pages)
    got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
    n = b.n_live
    far = ((got - want).abs() - bound - 1e-30)[:n]
    worst = far.flatten().argmax() if n else 0
    assert not torch.any(torch.isnan(got[:n]))
    assert torch.all(far <= 0), (float(far.max()), int(worst))
    assert torch.all(out[:, heads * b.dim:] == 7.0), "written behind a row"
    assert torch.all(out[n:] == 7.0), "written behind the last sequence"


ATTN = {
    "one token": dict(seqs=[(1, 1)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "one token 2": dict(seqs=[(1, 2)], heads=4, kv=1, dim=64, page=16, ty=rlh.F16),
    "decode 777": dict(seqs=[(1, 777)], heads=16, kv=8, dim=128, page=16, ty=rlh.BF16),
    "decode edges": dict(seqs=[(1, n) for n in (1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513)],
                         heads=8, kv=2, dim=128, page=32, ty=rlh.F16, pad_seqs=2, pad_rows=3),
    "decode ragged": dict(seqs=[(1, 5000), (1, 3), (0, 100), (1, 1200), (1, 64), (0, 0), (1, 2049)], heads=28, kv=4,
                          dim=128, page=64, ty=rlh.BF16),
    "decode 64": dict(seqs=[(1, 900 + 37 * i) for i in range(9)], heads=5, kv=1, dim=64, page=16, ty=rlh.BF16),
    "decode many": dict(seqs=[(1, 1 + (i * 37) % 300) for i in range(300)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16),
    "decode 16 per head": dict(seqs=[(1, 1500), (1, 31)], heads=32, kv=2, dim=128, page=128, ty=rlh.F16),
    "decode 24 per head": dict(seqs=[(1, 1500), (2, 31)], heads=24, kv=1, dim=128, page=16, ty=rlh.BF16),
    "decode long": dict(seqs=[(1, 30011), (1, 9)], heads=8, kv=1, dim=128, page=256, ty=rlh.BF16),
    "drafts": dict(seqs=[(4, 1300), (3, 3), (2, 65), (4, 4)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16),
    "prompt 1 2 3": dict(seqs=[(1, 1), (2, 2), (3, 3), (65, 65)], heads=4, kv=4, dim=128, page=16, ty=rlh.BF16),
    "prompt 517": dict(seqs=[(517, 517)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16),
    "prompt 1000 f16": dict(seqs=[(1000, 1000)], heads=4, kv=1, dim=64, page=64, ty=rlh.F16),
    "prompts": dict(seqs=[(129, 129), (64, 200), (0, 7), (128, 128), (31, 900), (1, 400)], heads=10, kv=2, dim=128, page=32,
                    ty=rlh.F16, pad_seqs=1, pad_rows=5),
    "chunk after long": dict(seqs=[(40, 6000)], heads=8, kv=1, dim=128, page=64, ty=rlh.BF16),
    "mixed": dict(seqs=[(300, 700), (1, 2000), (1, 1), (77, 77), (1, 515)], heads=32, kv=8, dim=128, page=16, ty=rlh.BF16),
    "cap": dict(seqs=[(70, 300), (1, 900)], heads=8, kv=4, dim=128, page=16, ty=rlh.BF16, cap=5.0, q_scale=6.0),
    "cap 64": dict(seqs=[(1, 333), (1, 2)], heads=8, kv=8, dim=64, page=32, ty=rlh.F16, cap=30.0, q_scale=6.0),
    "bias": dict(seqs=[(70, 300), (1, 900), (1, 1)], heads=12, kv=4, dim=128, page=16, ty=rlh.F16, bias=True),
    "bias long": dict(seqs=[(1, 20000)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, bias=True),
    "window": dict(seqs=[(200, 1000), (1, 900), (1, 5), (1, 64)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, window=64),
    "window 1": dict(seqs=[(33, 100), (1, 900)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16, window=1),
    "window 100 decode": dict(seqs=[(1, 5000), (1, 101), (1, 100), (1, 99)], heads=8, kv=2, dim=128, page=64, ty=rlh.F16,
                              window=100),
    "prefix": dict(seqs=[(100, 100), (200, 260), (1, 300), (5, 5)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16,
                   prefix=[37, 129, 12, 0]),
    "prefix past the end": dict(seqs=[(100, 100), (3, 3)], heads=4, kv=2, dim=128, page=16, ty=rlh.F16, prefix=[100000, 2]),
    "prefix window": dict(seqs=[(150, 400), (1, 600), (2, 600)], heads=4, kv=2, dim=128, page=16, ty=rlh.F16, window=50,
                          prefix=[100, 30, 599]),
    "everything": dict(seqs=[(150, 400), (1, 600), (9, 9)], heads=6, kv=2, dim=64, page=16, ty=rlh.BF16, window=70, bias=True,
                       cap=8.0, prefix=[20, 100, 9], q_scale=3.0),
    "shared": dict(seqs=[(1, 512 + i * 13 + 1) for i in range(20)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, shared=512),
    "shared only": dict(seqs=[(1, 65), (1, 64), (1, 70)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=64),
    "shared drafts": dict(seqs=[(3, 300), (1, 257), (30, 400), (2, 258)], heads=16, kv=2, dim=128, page=32, ty=rlh.F16,
                          shared=256),
    "shared long": dict(seqs=[(1, 8192 + 9 * i + 1) for i in range(5)], heads=16, kv=2, dim=64, page=64, ty=rlh.BF16,
                        shared=8192),
    "shared and shorter": dict(seqs=[(1, 20), (1, 500), (5, 200), (3, 3), (0, 9), (140, 300)], heads=8, kv=2, dim=128, page=16,
                               ty=rlh.BF16, shared=256, pad_rows=2),
    "shared window": dict(seqs=[(1, 700), (2, 530), (1, 513)], heads=8, kv=2, dim=128, page=16, ty=rlh.F16, shared=512,
                          window=100),
    "shared everything": dict(seqs=[(1, 700), (2, 530), (20, 533)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16, shared=512,
                              bias=True, cap=10.0, prefix=[600, 529, 100], window=300),
}


@pytest.mark.parametrize("name", list(ATTN))
def test_attention(name):
    case = dict(ATTN[name])
    heads = case["heads"]
    print("attention", name, case, flush=True)
    b, q, out, opts = attn_case(seed=len(name), **case)
    st = status_word()
    run_attn(b, q, out, heads, status=st, **opts)
    torch.cuda.synchronize()
    assert int(st) == 0
    check_attn(b, q, out, heads, opts)


MASKED = ["decode edges", "prompts", "mixed", "window", "prefix window", "shared and shorter", "drafts"]


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", MASKED)
def test_attention_ignores_what_no_row_may_see(name, fill):
    """Slots that no sequence holds (behind a length, inside a page) hold NaN
    or infinity."""
    case = dict(ATTN[name])
    b, q, out, opts = attn_case(seed=5, fill=fill, **case)
    run_attn(b, q, out, case["heads"], **opts)
    torch.cuda.synchronize()
    check_attn(b, q, out, case["heads"], opts)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["drafts", "prompts", "window", "prefix", "shared drafts"])
def test_attention_values_that_only_some_rows_see(name, bad):
    """K and V of one position are not finite: rows that do not see it are as
    if it were not there, rows that see it get NaN or that infinity."""
    case = dict(ATTN[name])
    heads = case["heads"]
    b, q, out, opts = attn_case(seed=6, **case)
    s = 0
    rows, n = case["seqs"][0]
    j = n - rows // 2 - 1
    keep = b.v[b.page_of(s, j), :, j % b.page].clone(), b.k[b.page_of(s, j), :, j % b.page].clone()
    b.v[b.page_of(s, j), :, j % b.page] = bad
    run_attn(b, q, out, heads, **opts)
    torch.cuda.synchronize()
    b.v[b.page_of(s, j), :, j % b.page] = keep[0]
    want, bound = ref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, b.dim ** -0.5, opts["cap"],
                                opts["slopes"], opts["window"], opts["prefix"])
    got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
    pos = torch.arange(n - rows, n, device="cuda")
    sees = pos >= j
    if opts["window"]:
        sees &= pos < j + opts["window"]
    if opts["prefix"] is not None:
        sees |= j < int(opts["prefix"][0])
    mine = torch.zeros(b.n_live, dtype=torch.bool, device="cuda")
    mine[:rows] = sees
    assert 0 < int(mine.sum()) < b.n_live
    hit = got[:b.n_live][mine]
    assert torch.all(torch.isnan(hit) if math.isnan(bad) else hit == bad)
    rest = ~mine
    assert torch.all((got[:b.n_live][rest] - want[:b.n_live][rest]).abs() <= bound[:b.n_live][rest] + 1e-30)
    # a NaN key: the rows that see it are NaN, the others as before
    b.k[b.page_of(s, j), :, j % b.page] = float("nan")
    run_attn(b, q, out, heads, **opts)
    torch.cuda.synchronize()
    got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
    assert torch.all(torch.isnan(got[:b.n_live][mine]))
    assert torch.all((got[:b.n_live][rest] - want[:b.n_live][rest]).abs() <= bound[:b.n_live][rest] + 1e-30)


def test_attention_infinite_scores():
    """Keys that give scores of minus infinity have no weight; where a row has
    no other, it is zero."""
    b, q, out, opts = attn_case([(1, 200), (40, 40)], 4, 2, 128, 16, rlh.BF16, seed=3)
    q[:, :4 * 128] = q[:, :4 * 128].abs() + 0.5
    for j in range(50, 120):
        b.k[b.page_of(0, j), :, j % 16] = -float("inf")
    for j in range(40):
        b.k[b.page_of(1, j), :, j % 16] = -float("inf")
    run_attn(b, q, out, 4, **opts)
    torch.cuda.synchronize()
    assert torch.all(out[1:41, :512] == 0)
    hidden = set()
    kk = b.k.clone()
    for j in range(50, 120):
        b.k[b.page_of(0, j), :, j % 16] = 0
    qr = q[:, :512].view(-1, 4, 128)
    # the plain form with those positions taken out
    k, v = b.rows_of(0)
    b.k = kk
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[50:120] = False
    for h in range(4):
        t = (qr[0, h].double() @ k[keep, h // 2].T) * 128 ** -0.5
        p = torch.softmax(t, 0)
        want = p @ v[keep, h // 2]
        near = p @ v[keep, h // 2].abs()
        tol = want.abs() * 2.0 ** -9 * 2 + near * (2.0 ** -8 + 2.0 ** -12)
        assert torch.all((out[0, h * 128:(h + 1) * 128].double() - want).abs() <= tol)
    assert not hidden


def test_attention_large_scores():
    """Scores of some thousands: the running maximum is taken over by later
    positions again and again (ascending keys)."""
    b, q, out, opts = attn_case([(1, 3000), (100, 700)], 8, 2, 128, 16, rlh.F16, seed=9, q_scale=20.0)
    for s, n in ((0, 3000), (1, 700)):
        for j in range(n):
            b.k[b.page_of(s, j), :, j % 16] *= 0.1 + 3.0 * j / n
    run_attn(b, q, out, 8, **opts)
    torch.cuda.synchronize()
    check_attn(b, q, out, 8, opts)


@pytest.mark.parametrize("name", ["decode ragged", "mixed", "shared drafts"])
def test_attention_pages_that_do_not_exist(name):
    """Positions in pages >= n_pages count as masked, and the status says so."""
    case = dict(ATTN[name])
    heads = case["heads"]
    b, q, out, opts = attn_case(seed=7, **case)
    st = status_word()
    victim = 0
    c = case.get("shared", 0) // b.page
    hidden = {b.page_of(victim, c * b.page)}
    b.table[victim, c] = -1
    run_attn(b, q, out, heads, status=st, **opts)
    torch.cuda.synchronize()
    assert int(st) == rlh.SERVE_BAD_PAGE
    check_attn(b, q, out, heads, opts, hidden)
    if case.get("shared"):
        st.zero_()
        hidden.add(b.shared_pages[1])
        b.shared_table[1] = b.n_pages + 5
        run_attn(b, q, out, heads, status=st, **opts)
        torch.cuda.synchronize()
        assert int(st) == rlh.SERVE_BAD_PAGE
        check_attn(b, q, out, heads, opts, hidden)


@pytest.mark.parametrize("name", ["decode ragged", "mixed", "shared drafts"])
def test_attention_skips_contradicting_sequences(name):
    case = dict(ATTN[name])
    heads = case["heads"]
    b, q, out, opts = attn_case(seed=8, **case)
    good = b.kv_len.clone()
    for wrong in (0, b.max_kv + 1, 0x7fffffff, -5):
        b.kv_len.copy_(good)
        b.kv_len[1] = wrong
        out.fill_(7.0)
        st = status_word()
        run_attn(b, q, out, heads, status=st, **opts)
        torch.cuda.synchronize()
        assert int(st) == rlh.SERVE_BAD_SEQ
        r0, r1 = int(b.starts[1]), int(b.starts[2])
        assert torch.all(out[r0:r1] == 7.0)
        want, bound = ref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, b.dim ** -0.5, opts["cap"],
                                    opts["slopes"], opts["window"], opts["prefix"])
        got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
        ok = torch.ones(b.n_rows, dtype=torch.bool, device="cuda")
        ok[r0:r1] = False
        assert torch.all((got - want).abs()[ok] <= bound[ok] + 1e-30)
    # starts that run past the rows: the last sequence is skipped
    b.kv_len.copy_(good)
    b.q_start[-1] = b.n_rows + 1000
    out.fill_(7.0)
    st = status_word()
    run_attn(b, q, out, heads, status=st, **opts)
    torch.cuda.synchronize()
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.all(out[int(b.starts[-2]):] == 7.0)


def test_attention_shared_prefix_equals_its_copies():
    """The same call with the prefix read through every sequence's own table."""
    case = dict(ATTN["shared drafts"])
    b, q, out, opts = attn_case(seed=4, **case)
    run_attn(b, q, out, case["heads"], **opts)
    b.table[:, :b.shared // b.page] = b.shared_table
    shared, b.shared = b.shared, 0
    out2 = torch.full_like(out, 7.0)
    b.shared_pages, keep = b.shared_pages, None
    run_attn(b, q, out2, case["heads"], **opts)
    torch.cuda.synchronize()
    b.shared = shared
    check_attn(b, q, out, case["heads"], opts)
    check_attn(b, q, out2, case["heads"], opts)


def test_attention_same_bits_every_time():
    for name in ("decode ragged", "mixed", "shared", "prompt 517"):
        case = dict(ATTN[name])
        b, q, out, opts = attn_case(seed=2, **case)
        run_attn(b, q, out, case["heads"], **opts)
        first = out.clone()
        for _ in range(3):
            out.fill_(7.0)
            run_attn(b, q, out, case["heads"], **opts)
            assert torch.equal(out, first)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 values: pages from its far end."""
    page, kv, dim = 256, 8, 128
    n_pages = (1 << 32) // (page * kv * dim) + 40
    b = ref.Batch([(1, 600), (70, 300)], kv, dim, page, rlh.BF16, seed=1)
    k = torch.zeros((n_pages, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros((n_pages, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    k[-b.n_pages:], v[-b.n_pages:] = b.k, b.v
    shift = n_pages - b.n_pages
    b.k, b.v, b.n_pages = k, v, n_pages
    b.table += torch.where(b.table < 0x7000000, shift, 0).to(torch.int32)
    b.table_host = np.where(b.table_host < 0x7000000, b.table_host + shift, b.table_host)
    g = torch.Generator().manual_seed(2)
    q = torch.randn((b.n_rows, 16 * dim), generator=g).to(torch.bfloat16).cuda()
    out = torch.full((b.n_rows, 16 * dim), 7.0, dtype=torch.bfloat16, device="cuda")
    run_attn(b, q, out, 16)
    torch.cuda.synchronize()
    check_attn(b, q, out, 16, dict(cap=0.0, slopes=None, window=0, prefix=None))
    x = append_inputs(b, 16, rlh.BF16, 4)
    run_append(b, x, rlh.BF16, 16, out, None, None, None, 1.0, 0, False)
    torch.cuda.synchronize()
    xs = x.view(b.n_rows, 32, dim)
    for s, (rows, n) in enumerate(b.seqs):
        for i in (0, rows - 1):
            p, r = n - rows + i, int(b.starts[s]) + i
            assert torch.equal(b.k[b.page_of(s, p), :, p % page], xs[r, 16:24])
            assert torch.equal(b.v[b.page_of(s, p), :, p % page], xs[r, 24:32])


# ---- sampling -------------------------------------------------------------------

def options_tensor(rows):
    raw = b"".join(bytes(rlh.RowSampling(*r)) for r in rows)
    return torch.frombuffer(bytearray(raw), dtype=torch.uint8).cuda()


def run_sample(logits, ty, rows, u, n=None, ws=None, st=None):
    n_rows = logits.shape[0]
    n = logits.shape[1] if n is None else n
    opt = options_tensor(rows)
    uu = torch.tensor(u, dtype=torch.float32, device="cuda")
    tok = torch.full((n_rows + 1,), -1, dtype=torch.int32, device="cuda")
    need = rlh.sample_rows_workspace(n_rows, n)
    if ws is None:
        ws = torch.full((need + 16,), 0xff, dtype=torch.uint8, device="cuda")
    rlh.sample_rows(ty, logits.data_ptr(), n_rows, n, logits.stride(0), opt.data_ptr(), uu.data_ptr(), tok.data_ptr(),
                    ws.data_ptr(), ws.numel() // 16 * 16, stream() if st is None else st)
    torch.cuda.synchronize()
    assert int(tok[-1]) == -1
    return tok[:-1].cpu().numpy()


SETS = [(0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 100, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05),
        (1.3, 0, 1.0, 0.0), (0.9, 1000, 0.8, 0.02), (1.0, 1, 0.5, 0.0), (2.0, 5000, 0.999, 0.0), (0.5, 0, 1e-6, 0.0),
        (1.0, 7, 1.0, 1.0), (-1.0, 3, 0.5, 0.5), (5.0, 0, 0.5, 0.0), (100.0, 0, 0.97, 0.0), (0.01, 0, 0.99, 0.0),
        (1.0, 3, 0.0, 0.0), (1.0, 50, -1.0, 0.0), (1.0, 2, 1.5, 1.5)]


@pytest.mark.parametrize("ty", [rlh.F32, rlh.F16, rlh.BF16])
@pytest.mark.parametrize("n", [1, 2, 63, 1000, 4097, 50001, 151936])
def test_sample_rows(n, ty):
    g = torch.Generator().manual_seed(n + ty)
    rng = np.random.default_rng(n + ty)
    rows = [s for s in SETS for _ in range(2)]
    stride = n + 5
    x = 2.5 * torch.randn((len(rows), stride), generator=g)
    x = x.to(TORCH[ty]).cuda()
    u = rng.random(len(rows)).astype(np.float32)
    u[0], u[1] = 0.0, np.float32(1 - 2.0 ** -24)
    got = run_sample(x, ty, rows, u, n=n)
    host = x[:, :n].double().cpu().numpy()
    for r, opt in enumerate(rows):
        assert got[r] == ref.sample(host[r], *opt, u[r]), (r, opt, u[r])


def test_sample_ties():
    """Rows of few distinct values: the order of equal ones decides what top-k
    and top-p keep."""
    rng = np.random.default_rng(3)
    rows, us, xs = [], [], []
    for n_values in (1, 2, 5):
        for opt in [(1.0, 40, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (0.7, 1500, 0.31, 0.0), (1.0, 0, 1.0, 0.9), (1.0, 0, 1.0, 0.0),
                    (1.0, 3, 0.999, 0.0)]:
            for _ in range(3):
                xs.append(rng.integers(0, n_values, 3001).astype(np.float32) - 1.0)
                rows.append(opt)
                us.append(rng.random())
    x = torch.tensor(np.stack(xs)).cuda()
    u = np.array(us, np.float32)
    got = run_sample(x, rlh.F32, rows, u)
    for r, opt in enumerate(rows):
        assert got[r] == ref.sample(xs[r], *opt, u[r]), (r, opt)


def test_sample_special_values():
    nan, inf = float("nan"), float("inf")
    n = 2000
    base = np.linspace(-3, 3, n).astype(np.float32)
    xs = [base.copy() for _ in range(9)]
    xs[0][:] = -inf
    xs[1][:] = nan
    xs[2][5] = nan
    xs[2][1990:] = -inf
    xs[3][[100, 700]] = inf
    xs[4][:] = -inf
    xs[4][1234] = -2.0
    xs[5][:] = -np.finfo(np.float32).max
    xs[6][:] = 0.0
    xs[6][::2] = -0.0
    xs[7][:1000] = np.float32(3e38)
    xs[7][1000:] = np.float32(-3e38)
    xs[8][::3] = nan
    x = torch.tensor(np.stack(xs)).cuda()
    for opt in [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 3, 1.0, 0.1),
                (inf, 0, 1.0, 0.0), (nan, 0, 1.0, 0.0), (1.0, 0, nan, nan), (1e-30, 10, 0.9, 0.0)]:
        for u in (0.0, 0.37, 0.999):
            us = np.full(len(xs), u, np.float32)
            got = run_sample(x, rlh.F32, [opt] * len(xs), us)
            want = [ref.sample(v, opt[0], opt[1], 0.0 if math.isnan(opt[2]) else opt[2],
                               0.0 if math.isnan(opt[3]) else opt[3], np.float32(u)) for v in xs]
            assert list(got) == want, (opt, u)


def test_sample_u_outside_its_range():
    x = torch.tensor(np.linspace(-1, 1, 500, dtype=np.float32)[None].repeat(4, 0)).cuda()
    opt = [(1.0, 0, 1.0, 0.0)] * 4
    got = run_sample(x, rlh.F32, opt, np.array([-3.0, float("nan"), 1.0, 7.0], np.float32))
    assert list(got) == [0, 0, 499, 499]


# ---- a step as a server makes it --------------------------------------------------

def serve_step(b, x, heads, freqs, w, q_rows, out, logits_w, options, u, tok, ws, status, st):
    """Append, attention, a projection to logits, one token per row."""
    run_append(b, x, rlh.F32, heads, q_rows, w, w, freqs, 1.0, b.dim, False, status, st)
    run_attn(b, q_rows, out, heads, status=status, ws=ws, st=st)
    logits = out.float() @ logits_w
    n = logits.shape[1]
    rlh.sample_rows(rlh.F32, logits.data_ptr(), logits.shape[0], n, n, options.data_ptr(), u.data_ptr(), tok.data_ptr(),
                    ws.data_ptr(), ws.numel() // 16 * 16, st)
    return logits


@pytest.mark.parametrize("shared", [0, 64])
def test_a_step_captured_and_replayed(shared):
    """Append, attention and sampling on a stream of their own, captured once
    and replayed with other lengths, rows and random numbers, beside eager
    calls of the same operators; every replay equals the plain forms."""
    heads, kv, dim, page, vocab = 8, 2, 128, 16, 777
    lens = [90, 65, 200, 131]
    b = ref.Batch([(1, n + 8) for n in lens], kv, dim, page, rlh.F16, seed=11, shared=shared)
    b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
    b.max_kv = max(lens) + 8
    g = torch.Generator().manual_seed(5)
    w = (1 + 0.1 * torch.randn(dim, generator=g)).cuda()
    logits_w = torch.randn((heads * dim, vocab), generator=g).cuda()
    freqs = torch.tensor(rlh.rope_freqs(dim, 1e6)[0]).cuda()
    x = torch.zeros((4, (heads + 2 * kv) * dim), device="cuda")
    q_rows = torch.zeros((4, heads * dim), dtype=torch.float16, device="cuda")
    out = torch.zeros((4, heads * dim), dtype=torch.float16, device="cuda")
    options = options_tensor([(0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0)])
    u = torch.zeros(4, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    status = status_word()
    ws = torch.full((64 << 20,), 0xff, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        logits_w @ torch.zeros((vocab, 1), device="cuda")  # the product's library is loaded before the capture
        out.float() @ logits_w
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            logits = serve_step(b, x, heads, freqs, w, q_rows, out, logits_w, options, u, tok, ws, status,
                                side.cuda_stream)
    torch.cuda.synchronize()
    rng = np.random.default_rng(7)
    opts = [(0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0)]
    for step in range(5):
        now = [n + step for n in lens]
        b.seqs = [(1, n) for n in now]
        b.kv_len.copy_(torch.tensor(now, dtype=torch.int32))
        x.copy_(1.5 * torch.randn(x.shape, generator=g))
        uu = rng.random(4).astype(np.float32)
        u.copy_(torch.tensor(uu))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0
        qe, ke, ve, q_off, k_off, _ = append_expected(b, x, heads, w, w, freqs, 1.0, dim, False)
        h2 = half(rlh.F16)
        assert torch.all((q_rows.double().view(4, heads, dim) - qe).abs() <= qe.abs() * h2 + 2 * q_off + 2.0 ** -25)
        for s, n in enumerate(now):
            got = b.k[b.page_of(s, n - 1), :, (n - 1) % page].double()
            assert torch.all((got - ke[s]).abs() <= ke[s].abs() * h2 + 2 * k_off[s] + 2.0 ** -25)
            assert torch.equal(b.v[b.page_of(s, n - 1), :, (n - 1) % page], ve[s].half())
        want, bound = ref.attention(b, q_rows.view(4, heads, dim), heads, dim ** -0.5)
        assert torch.all((out.double().view(4, heads, dim) - want).abs() <= bound + 1e-30)
        host = logits.double().cpu().numpy()
        assert [int(t) for t in tok.cpu()] == [ref.sample(host[r], *opts[r], uu[r]) for r in range(4)]
        # the program's own eager calls between the replays
        eager = torch.full_like(out, 7.0)
        run_attn(b, q_rows, eager, heads)
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


def test_two_streams_with_workspaces_of_their_own():
    case = dict(ATTN["decode ragged"])
    jobs = []
    for i in range(2):
        b, q, out, opts = attn_case(seed=20 + i, **case)
        jobs.append((b, q, out, opts, torch.cuda.Stream()))
    torch.cuda.synchronize()
    keep = []
    for _ in range(10):
        for b, q, out, opts, s in jobs:
            with torch.cuda.stream(s):
                keep.append(run_attn(b, q, out, case["heads"], st=s.cuda_stream, **opts))
    torch.cuda.synchronize()
    for b, q, out, opts, _ in jobs:
        check_attn(b, q, out, case["heads"], opts)


def test_refused_on_the_device():
    """Host memory, and a workspace that is too small."""
    b, q, out, opts = attn_case([(1, 3000)], 8, 2, 128, 16, rlh.BF16)
    host = np.zeros(1 << 16, np.uint8)
    lib = rlh.load()
    args = rlh.AttnArgs(8, 0, q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0), 0.1, 0.0, None, None, None, 0)
    ws = torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    bad_q = rlh.AttnArgs(8, 0, (host.ctypes.data + 15) // 16 * 16, out.data_ptr(), q.stride(0), out.stride(0), 0.1, 0.0,
                         None, None, None, 0)
    kv, seqs = b.kv(), b.desc()
    assert lib.rlh_paged_attn(kv, seqs, bad_q, ws.data_ptr(), ws.numel(), None, None) == rlh.RLH_EINVAL
    assert b"device-accessible" in lib.rlh_last_error()
    assert lib.rlh_paged_attn(kv, seqs, args, ws.data_ptr(), ws.numel(), host.ctypes.data // 4 * 4, None) == rlh.RLH_EINVAL
    need = rlh.paged_attn_workspace(kv, seqs, args)
    if need:
        assert lib.rlh_paged_attn(kv, seqs, args, ws.data_ptr(), need - 1, None, None) == rlh.RLH_EINVAL
        assert b"workspace" in lib.rlh_last_error()
    torch.cuda.synchronize()
    assert torch.all(out == 7.0)


# ---- divisions of the work, scales, long rows --------------------------------------

ATTN_MORE = {
    # 320 rows of a KV head: a whole tile and one of 64 rows, divided into fewer parts
    "shared uneven": dict(seqs=[(4, 4608 + 4 + i) for i in range(20)], heads=32, kv=8, dim=64, page=64, ty=rlh.BF16,
                          shared=4608),
    "shared uneven all masks": dict(seqs=[(4, 4608 + 4 + 7 * i) for i in range(20)], heads=32, kv=8, dim=64, page=64,
                                    ty=rlh.F16, shared=4608, cap=10.0, bias=True, window=2000, prefix=[300 * i for i in range(20)]),
    # a bias that grows with positions behind a row's own
    "prefix bias": dict(seqs=[(300, 300), (70, 500), (1, 700)], heads=8, kv=4, dim=128, page=16, ty=rlh.BF16, bias=True,
                        prefix=[250, 499, 700]),
    "cap and bias": dict(seqs=[(100, 1100), (1, 1500)], heads=12, kv=4, dim=128, page=32, ty=rlh.F16, bias=True, cap=4.0,
                         q_scale=4.0),
    # short sequences: one block each, or (more blocks than run at once) divided
    "decode short": dict(seqs=[(1, 1 + (i * 37) % 500) for i in range(40)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16),
    "decode many short": dict(seqs=[(1, 1 + (i * 37) % 250) for i in range(140)], heads=8, kv=2, dim=128, page=16, ty=rlh.BF16),
    "decode many shorter": dict(seqs=[(1, 1 + (i * 37) % 128) for i in range(140)], heads=8, kv=2, dim=64, page=32, ty=rlh.F16),
    "mixed with drafts": dict(seqs=[(300, 310), (2, 900), (1, 33), (4, 4), (0, 5), (90, 2000)], heads=16, kv=4, dim=64, page=16,
                              ty=rlh.F16, pad_seqs=2, pad_rows=4),
}


@pytest.mark.parametrize("name", list(ATTN_MORE))
def test_attention_more(name):
    case = dict(ATTN_MORE[name])
    heads = case["heads"]
    print("attention", name, case, flush=True)
    b, q, out, opts = attn_case(seed=len(name), **case)
    st = status_word()
    run_attn(b, q, out, heads, status=st, **opts)
    torch.cuda.synchronize()
    assert int(st) == 0
    check_attn(b, q, out, heads, opts)


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 0.3])
@pytest.mark.parametrize("name", ["decode ragged", "mixed", "cap", "bias", "shared drafts"])
def test_attention_scales(name, scale):
    case = dict(ATTN[name])
    heads = case["heads"]
    b, q, out, opts = attn_case(seed=13, **case)
    run_attn(b, q, out, heads, scale=scale, **opts)
    torch.cuda.synchronize()
    want, bound = ref.attention(b, q[:, :heads * b.dim].view(-1, heads, b.dim), heads, scale, opts["cap"], opts["slopes"],
                                opts["window"], opts["prefix"])
    got = out[:, :heads * b.dim].double().view(-1, heads, b.dim)
    assert torch.all((got - want).abs()[:b.n_live] <= bound[:b.n_live] + 1e-30)


@pytest.mark.parametrize("ty", [rlh.F32, rlh.F16, rlh.BF16])
@pytest.mark.parametrize("n,shift", [(300001, 0), (300001, 1), (163841, 3), (131072, 0)])
def test_sample_long_rows(n, shift, ty):
    """More groups of 64 than are held or listed at a time; rows that begin
    inside a 16-byte line."""
    rows = [(1.0, 0, 0.9, 0.0), (20.0, 0, 0.9, 0.0), (1.0, 1000, 0.99, 0.0), (1.5, 20000, 1.0, 0.0), (1.0, 0, 1.0, 1e-4),
            (1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0)]
    g = torch.Generator().manual_seed(n + ty + shift)
    x = 2.0 * torch.randn((len(rows), n + 9), generator=g)
    x = x.to(TORCH[ty]).cuda()[:, shift:]
    u = np.random.default_rng(n + ty).random(len(rows)).astype(np.float32)
    got = run_sample(x, ty, rows, u, n=n)
    host = x[:, :n].double().cpu().numpy()
    for r, opt in enumerate(rows):
        assert got[r] == ref.sample(host[r], *opt, u[r]), (r, opt, u[r])


def test_sample_long_ties():
    """Many more equal values than are held, over all groups, and a border in
    the middle of them."""
    n = 200003
    xs, rows, us = [], [], []
    for opt in [(1.0, 1000, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, 150000, 0.5, 0.0), (1.0, 0, 1.0, 1.0), (0.5, 700, 0.8, 0.5),
                (1.0, 0, 1.0, 0.0)]:
        for kind in range(3):
            v = np.zeros(n, np.float32)
            if kind == 1:
                v[::2] = -1.0
            if kind == 2:
                v[:] = -np.inf
                v[5::3] = 4.0
                v[100::1000] = 4.5
            xs.append(v)
            rows.append(opt)
            us.append(0.123 + 0.04 * len(us))
    u = np.array(us, np.float32)
    got = run_sample(torch.tensor(np.stack(xs)).cuda(), rlh.F32, rows, u)
    for r, opt in enumerate(rows):
        assert got[r] == ref.sample(xs[r], *opt, u[r]), (r, opt)


def test_sample_longest_row():
    n = 1 << 21
    g = torch.Generator().manual_seed(1)
    x = (3.0 * torch.randn((4, n), generator=g)).half().cuda()
    rows = [(1.0, 0, 0.9, 0.0), (1.0, 50, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (0.8, 5000, 0.99, 1e-5)]
    u = np.array([0.3, 0.6, 0.9, 0.99], np.float32)
    got = run_sample(x, rlh.F16, rows, u)
    host = x.double().cpu().numpy()
    for r, opt in enumerate(rows):
        assert got[r] == ref.sample(host[r], *opt, u[r]), (r, opt)


def test_append_with_starts_that_fall():
    """A row that lies in no sequence, though the starts name one by their
    count: left as it was, and the status says so."""
    b = ref.Batch([(5, 40), (5, 40), (5, 40)], 2, 128, 16, rlh.F16, seed=3)
    b.q_start.copy_(torch.tensor([0, 30, 5, 10], dtype=torch.int32)[:b.q_start.numel()])
    x = append_inputs(b, 4, rlh.F32, 5)
    q_out = torch.full((b.n_rows, 4 * 128), 7.0, dtype=torch.float16, device="cuda")
    k = b.k.clone()
    st = status_word()
    run_append(b, x, rlh.F32, 4, q_out, None, None, None, 1.0, 0, False, st)
    torch.cuda.synchronize()
    assert int(st) == rlh.SERVE_BAD_SEQ
    assert torch.all(q_out[10:] == 7.0) and torch.all(q_out[:5] == 7.0)
    changed = torch.any(torch.any(b.k != k, dim=3), dim=1)
    assert int(changed.sum()) <= 5


# ---- more sequences than a wave looks at by itself -----------------------------------

ATTN_MANY = {
    "tokens": dict(seqs=[(1, 1 + (i * 61) % 700) for i in range(1100)], heads=4, kv=2, dim=64, page=16, ty=rlh.F16),
    "tokens short": dict(seqs=[(1, 1 + (i * 37) % 128) for i in range(259)], heads=2, kv=1, dim=64, page=16, ty=rlh.BF16),
    "tokens and prompts": dict(seqs=[((0, 1, 20, 2)[i % 4], 30 + (i * 37) % 300) for i in range(300)] + [(300, 310)], heads=8,
                               kv=2, dim=64, page=16, ty=rlh.BF16, pad_seqs=3, pad_rows=2),
    "wide groups": dict(seqs=[(1, 1 + (i * 37) % 200) for i in range(280)], heads=20, kv=1, dim=64, page=32, ty=rlh.F16),
    "shared": dict(seqs=[(1 + i % 7 // 6 * 8, 80 + (i * 37) % 200) for i in range(270)], heads=4, kv=1, dim=64, page=16,
                   ty=rlh.F16, shared=64),
}


@pytest.mark.parametrize("name", list(ATTN_MANY))
def test_attention_many_sequences(name):
    case = dict(ATTN_MANY[name])
    heads = case["heads"]
    print("attention", name, flush=True)
    b, q, out, opts = attn_case(seed=len(name), **case)
    st = status_word()
    run_attn(b, q, out, heads, status=st, **opts)
    torch.cuda.synchronize()
    assert int(st) == 0
    check_attn(b, q, out, heads, opts)
    # one that contradicts the bounds
    b.kv_len[260 % len(case["seqs"])] = b.max_kv + 1
    run_attn(b, q, torch.empty_like(out), heads, status=st, **opts)
    torch.cuda.synchronize()
    rows = case["seqs"][260 % len(case["seqs"])][0]
    assert int(st) == (rlh.SERVE_BAD_SEQ if rows else 0)


def test_append_many_sequences():
    seqs = [((0, 1, 3, 1)[i % 4], 5 + (i * 37) % 90) for i in range(600)]
    b = ref.Batch(seqs, 1, 64, 16, rlh.F16, seed=8, pad_seqs=2, pad_rows=3)
    x = append_inputs(b, 2, rlh.F16, 5)
    q_out = torch.full((b.n_rows, 2 * 64), 7.0, dtype=torch.float16, device="cuda")
    st = status_word()
    run_append(b, x, rlh.F16, 2, q_out, None, None, None, 1.0, 0, False, st)
    torch.cuda.synchronize()
    assert int(st) == 0
    xs = x[:, :4 * 64].view(b.n_rows, 4, 64)
    assert torch.equal(q_out[:b.n_live], xs[:b.n_live, :2].reshape(-1, 128)) and torch.all(q_out[b.n_live:] == 7.0)
    for s, (rows, n) in enumerate(seqs):
        for i in range(rows):
            p, r = n - rows + i, int(b.starts[s]) + i
            assert torch.equal(b.k[b.page_of(s, p), :, p % 16], xs[r, 2:3])
            assert torch.equal(b.v[b.page_of(s, p), :, p % 16], xs[r, 3:4])
