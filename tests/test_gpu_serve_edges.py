"""Ends of the ranges that the batched serving operators accept, on the GPU
against 64-bit forms."""
import ctypes

import numpy as np
import pytest
import torch

import rlh
import serve_ref as ref
from test_gpu_serve import (ATTN, append_inputs, attn_case, check_attn, options_tensor, run_append, run_attn,
                            run_sample)

pytestmark = pytest.mark.gpu

TORCH = ref.TORCH


def compare_samples(xs, rows, us, ty=rlh.F32, shift=0):
    """Rows that begin `shift` values into a 16-byte line."""
    n = len(xs[0])
    width = (n + shift + 15) // 16 * 16
    x = torch.zeros((len(xs), width), dtype=TORCH[ty])
    x[:, shift:shift + n] = torch.tensor(np.stack(xs)).to(TORCH[ty])
    host = x[:, shift:shift + n].double().numpy()
    got = run_sample(x.cuda()[:, shift:], ty, rows, np.array(us, np.float32), n=n)
    want = [ref.sample(host[r], *rows[r], np.float32(us[r])) for r in range(len(xs))]
    wrong = [(r, int(g), w, rows[r], us[r]) for r, (g, w) in enumerate(zip(got, want)) if int(g) != w]
    assert not wrong, wrong[:8]


FILTERS = [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (1.0, 1500, 1.0, 0.0), (1.0, 40, 1.0, 0.0),
           (1.0, 40, 0.9, 0.0), (0.1, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("ty", [rlh.F32, rlh.F16, rlh.BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_sample_past_the_draw_with_a_tail_of_no_weight(shift, ty):
    """u of 1 and more takes the last kept token that has weight, though whole
    chunks behind it have (next to) none, and the first logit is -infinity."""
    rng = np.random.default_rng(shift)
    xs, rows, us = [], [], []
    for depth in (28.0, 50.0, 120.0, 300.0, 1000.0):
        for opt in FILTERS:
            for u in (1.0, 7.0, 1 - 2.0 ** -24):
                v = np.full(9000, -depth, np.float32) + rng.random(9000).astype(np.float32)
                v[:4096] = rng.random(4096)
                v[0] = -np.inf
                xs.append(v)
                rows.append(opt)
                us.append(u)
    compare_samples(xs, rows, us, ty, shift)


@pytest.mark.parametrize("shift", [0, 1])
def test_sample_past_the_draw_at_low_temperature(shift):
    rng = np.random.default_rng(7)
    n = 151936
    xs, rows, us = [], [], []
    for temperature in (0.05, 0.1, 0.2, 0.7):
        for u in (1.0, 3.0):
            v = (2.2 * rng.standard_normal(n)).astype(np.float32)
            v[rng.integers(0, n, 24)] = 7 + 5 * rng.random(24)
            xs.append(v)
            rows.append((temperature, 0, 1.0, 0.0))
            us.append(u)
    compare_samples(xs, rows, us, shift=shift)


def test_sample_inside_a_chunk_of_little_weight():
    """u that falls into the first chunk, whose weights are e^-60 of the rest's."""
    w = np.exp(-60.0)
    xs, rows, us = [], [], []
    for at in (0.0, 0.5, 1000.5, 4094.5):
        v = np.zeros(9000, np.float32)
        v[:4096] = -60.0
        xs.append(v)
        rows.append((1.0, 0, 1.0, 0.0))
        us.append(at * w / 4904.0)
    compare_samples(xs, rows, us)


# ---- borders far below the largest weight ------------------------------------------

DEEP = [(1.0, 2000, 1.0, 0.0), (1.0, 5000, 1.0, 0.0), (1.0, 0, 1.0, 4e-13), (1.0, 3000, 1.0, 5e-13), (0.5, 2000, 1.0, 0.0),
        (1.0, 5999, 1.0, 0.0), (2.0, 2000, 1.0, 0.0)]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("kind", ["spread", "equal", "steps"])
def test_sample_borders_below_the_histograms(kind, shift):
    """One likely token, and thousands at some 2^-41 of it among which top-k
    or min-p ends."""
    rng = np.random.default_rng(11)
    n = 6000 if kind == "spread" else 20000
    xs, rows, us = [], [], []
    for opt in DEEP:
        for u in (1.0, 1 - 2.0 ** -24, 0.3):
            v = rng.normal(-28.4, 0.3, n).astype(np.float32)
            if kind == "equal":
                v[:] = -28.4
            if kind == "steps":
                v = np.round(v * 8) / 8
            v *= opt[0]
            v[rng.integers(0, n)] = 0.0
            xs.append(v.astype(np.float32))
            rows.append(opt)
            us.append(u)
    compare_samples(xs, rows, us, shift=shift)


def test_sample_long_flat_row_behind_one_token():
    """151936 logits, one 28 above the rest: what top-k leaves is less than a
    step of u away from 1, the whole rest is more."""
    n = 151936
    xs, rows, us = [], [], []
    for k in (1200, 2000, 30000):
        v = np.zeros(n, np.float32)
        v[0] = 28.0
        xs.append(v)
        rows.append((1.0, k, 1.0, 0.0))
        us.append(1 - 2.0 ** -24)
    compare_samples(xs, rows, us)


def test_sample_draws_in_a_deep_tail():
    """The draw falls among tokens of 2^-40.4 of the largest: inside the first
    top_k, and where 64 bits put it as far as the masses go, 2^-37 of the
    largest: 11 tokens."""
    n = 1 << 18
    v = np.full(n, -28.0, np.float32)
    v[0] = 0.0
    k = 120000
    u = np.full(2, 1 - 2.0 ** -24, np.float32)
    got = run_sample(torch.tensor(np.stack([v, v])).cuda(), rlh.F32, [(1.0, k, 1.0, 0.0)] * 2, u)
    want = ref.sample(v, 1.0, k, 1.0, 0.0, u[0])
    assert 0 < want < k and abs(int(got[1]) - want) <= 11


def test_sample_nucleus_that_ends_deep():
    """top-p that ends among equal tokens of 2^-40.4 of the largest: the last
    kept one is where 64 bits put it to 2^-36 of the mass, 21 tokens."""
    n = 1 << 18
    v = np.full(n, -28.0, np.float32)
    v[5] = 0.0
    p = np.float32(1 - 2.0 ** -23)
    got = run_sample(torch.tensor(np.stack([v, v])).cuda(), rlh.F32, [(1.0, 0, p, 0.0)] * 2, np.ones(2, np.float32))
    want = ref.sample(v, 1.0, 0, p, 0.0, np.float32(1.0))
    assert 1000 < want < n - 1000 and abs(int(got[1]) - want) <= 21


# ---- attention: caps, flat rows ------------------------------------------------------

class Shared:
    """`n_seq` sequences of `rows` new rows whose pages are the same ones."""

    def __init__(self, k, v, n_seq, rows, heads, ty, page=64):
        n, kv, dim = k.shape
        pages = -(-n // page)
        pool = torch.zeros((2, pages * page, kv, dim), dtype=torch.float64)
        pool[0, :n], pool[1, :n] = k, v
        pool = pool.view(2, pages, page, kv, dim).transpose(2, 3).contiguous().to(TORCH[ty]).cuda()
        self.k, self.v, self.heads, self.dim, self.rows, self.n, self.kv_heads = pool[0], pool[1], heads, dim, rows, n, kv
        self.table = torch.arange(pages, dtype=torch.int32).repeat(n_seq, 1).cuda()
        self.q_start = (rows * torch.arange(n_seq + 1, dtype=torch.int32)).cuda()
        self.kv_len = torch.full((n_seq,), n, dtype=torch.int32).cuda()
        self.kv = rlh.KvPages(ty, kv, dim, page, pages, self.k.data_ptr(), self.v.data_ptr())
        self.seqs = rlh.Seqs(n_seq, n_seq * rows, rows, n, pages, self.q_start.data_ptr(), self.kv_len.data_ptr(),
                             self.table.data_ptr())

    def run(self, q, scale, cap=0.0):
        out = torch.full_like(q, 7.0)
        args = rlh.AttnArgs(self.heads, 0, q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0), scale, cap, None, None,
                            None, 0)
        need = rlh.paged_attn_workspace(self.kv, self.seqs, args)
        ws = torch.full((need + 16,), 0xff, dtype=torch.uint8, device="cuda")
        rlh.paged_attn(self.kv, self.seqs, args, ws.data_ptr(), ws.numel() // 16 * 16, None,
                       torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out


U = 2.0 ** -24


@pytest.mark.parametrize("cap", [65.0, 1e3, 1e5, 1e8, 1e30, 3.4e38])
@pytest.mark.parametrize("size", [1.0, 40.0])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_caps_far_above_the_scores(rows, size, cap):
    """tanh's relative error counts, not the cap's: a score is off by what
    the dot product is, (dim + 8) 2^-24 sum |q k|, and 16 half steps of its own
    size for the cap's terms and the exponent's argument. That scales a
    probability once in the sum with v and once in the sum below it; the rest
    is the probabilities' rounding (of the smallest: to multiples of 2^-24), f32
    sums of n terms and the result's rounding."""
    n, heads, kv, dim, ty = 300, 4, 2, 128, rlh.F16
    g = torch.Generator().manual_seed(rows)
    k, v = [torch.randn((n, kv, dim), generator=g).half().double() for _ in range(2)]
    q = (size * torch.randn((rows, heads * dim), generator=g)).half()
    scale = float(np.float32(dim ** -0.5))
    out = Shared(k, v, 1, rows, heads, ty).run(q.cuda(), scale, cap).double().cpu().view(rows, heads, dim)
    cap = float(np.float32(cap))
    see = torch.arange(n)[None, :] <= torch.arange(n - rows, n)[:, None]
    half = torch.finfo(torch.float16).eps / 2
    for h in range(heads):
        qh, kh, vh = q.double().view(rows, heads, dim)[:, h], k[:, h // 2], v[:, h // 2]
        t = scale * (qh @ kh.T)
        ds = ((dim + 8) * U * scale * (qh.abs() @ kh.abs().T) + 16 * U * t.abs()).amax(1, keepdim=True)
        p = torch.softmax(torch.where(see, cap * torch.tanh(t / cap), -float("inf")), 1)
        want, near = p @ vh, p @ vh.abs()
        bound = want.abs() * half + near * (half + 2 * (ds + n * U)) + 2.0 ** -25 * (see.double() @ vh.abs())
        assert torch.all((out[:, h] - want).abs() <= bound), (h, float(((out[:, h] - want).abs() / bound).max()))


@pytest.mark.parametrize("cap", [65.0, 1e4])
@pytest.mark.parametrize("name", ["everything", "shared everything", "cap 64", "mixed", "decode ragged", "bias", "shared"])
def test_attention_larger_caps(name, cap):
    """Caps above 64 beside every mask, type and head size."""
    case = dict(ATTN[name], cap=cap, q_scale=12.0)
    b, q, out, opts = attn_case(seed=21, **case)
    run_attn(b, q, out, case["heads"], **opts)
    torch.cuda.synchronize()
    check_attn(b, q, out, case["heads"], opts)


@pytest.mark.parametrize("top", ["first", "last"])
@pytest.mark.parametrize("n_seq,rows,kv", [(100, 1, 8), (20, 64, 8)])
def test_attention_flat_rows_in_f16(n_seq, rows, kv, top):
    """One score 17.5 above thousands of equal ones: each has less than 2^-25
    of its weight, all of them what counts (the first's value is zero).
    The result is off by its own rounding, by f32's sums, and by what half a step of
    f16's smallest, 2^-25, is of probabilities of up to 2^7 and more: 2^-32 a position."""
    n, dim, group = 20000, 128, 4
    k = torch.zeros((n, kv, dim), dtype=torch.float64)
    v = torch.ones((n, kv, dim), dtype=torch.float64)
    at = 0 if top == "first" else n - rows
    k[at, :, 0] = 17.5
    v[at] = 0.0
    q = torch.zeros((n_seq * rows, kv * group, dim), dtype=torch.float16)
    q[:, :, 0] = 8.0
    b = Shared(k, v, n_seq, rows, kv * group, rlh.F16)
    out = b.run(q.view(n_seq * rows, -1).cuda(), 0.125).double().view(n_seq, rows, kv * group * dim)
    seen = torch.arange(n - rows, n, dtype=torch.float64, device="cuda")[None, :, None] + 1
    w = float(np.exp(-17.5))
    L = 1 + (seen - 1) * w
    want = (seen - 1) * w / L
    bound = want * (2.0 ** -11 + 2 * (40 + n) * U) + seen * 2.0 ** -32 / L + 2.0 ** -25
    assert torch.all((out - want).abs() <= bound), (float(out.min()), float(out.max()), float(want.min()))


def test_attention_one_workspace_for_limits():
    """Prompts, single tokens, drafts and a shared prefix in the workspace of a
    host's limits, one after the other."""
    heads, kv, dim, page, ty = 8, 2, 128, 16, rlh.BF16
    batches = [dict(seqs=[(700, 700)]), dict(seqs=[(1, 3000)]), dict(seqs=[(130, 2500), (1, 9)]), dict(seqs=[(4, 2000)] * 3),
               dict(seqs=[(1, 40)] * 30), dict(seqs=[(1, 1100 + i) for i in range(9)], shared=1024),
               dict(seqs=[(3, 1100), (40, 1500)], shared=1024), dict(seqs=[(200, 2999)])]
    first = attn_case(seed=1, heads=heads, kv=kv, dim=dim, page=page, ty=ty, **batches[5])[0]
    p = first.q_start.data_ptr()
    limits = rlh.Seqs(30, 700, 700, 3000, -(-3000 // page), p, p, p)
    args = rlh.AttnArgs(heads, 0, first.k.data_ptr(), first.v.data_ptr() + (1 << 40), heads * dim, heads * dim, 0.1, 0.0,
                        None, None, p, 1024)
    need = rlh.paged_attn_workspace(first.kv(), limits, args)
    assert 0 < need < 64 << 20
    guard = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device="cuda")
    ws = guard[:need]
    for i, batch in enumerate(batches):
        ws.fill_(0xff)
        b, q, out, opts = attn_case(seed=30 + i, heads=heads, kv=kv, dim=dim, page=page, ty=ty, **batch)
        run_attn(b, q, out, heads, ws=ws, **opts)
        torch.cuda.synchronize()
        check_attn(b, q, out, heads, opts)
    assert torch.all(guard[need:] == 0xa5)


# ---- errors of the caller's own ------------------------------------------------------

def test_errors_that_a_caller_left_are_not_a_calls_own():
    """A HIP error that the host caused before and has not asked for: the calls
    are enqueued and say so."""
    hip = ctypes.CDLL(rlh.LIB_PATH)  # (its symbols include those of the runtime that it is linked to)
    n = 5000
    x = torch.randn((2, n), generator=torch.Generator().manual_seed(1)).cuda()
    opt = options_tensor([(0.0, 0, 1.0, 0.0)] * 2)
    u = torch.zeros(2, device="cuda")
    tok = torch.full((2,), -1, dtype=torch.int32, device="cuda")
    ws = torch.empty(rlh.sample_rows_workspace(2, n), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    b = ref.Batch([(3, 20), (1, 700), (40, 40)], 2, 128, 16, rlh.BF16, seed=1)
    rows = append_inputs(b, 4, rlh.F32, 2)
    q = torch.randn((b.n_rows, 512), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    out, q_out = torch.zeros_like(q), torch.zeros_like(q)
    try:
        for call in (lambda: rlh.sample_rows(rlh.F32, x.data_ptr(), 2, n, n, opt.data_ptr(), u.data_ptr(), tok.data_ptr(),
                                             ws.data_ptr(), ws.numel(), st),
                     lambda: run_append(b, rows, rlh.F32, 4, q_out, None, None, None, 1.0, 0, False)):
            assert hip.hipSetDevice(-7) != 0
            call()
        args = rlh.AttnArgs(4, 0, q.data_ptr(), out.data_ptr(), 512, 512, 0.1, 0.0, None, None, None, 0)
        space = torch.empty(rlh.paged_attn_workspace(b.kv(), b.desc(), args) + 16, dtype=torch.uint8, device="cuda")
        assert hip.hipSetDevice(-7) != 0
        rlh.paged_attn(b.kv(), b.desc(), args, space.data_ptr(), space.numel() // 16 * 16, None, st)
    finally:
        hip.hipGetLastError()
    torch.cuda.synchronize()
    assert tok.cpu().tolist() == x.argmax(1).cpu().tolist()


# ---- tiny temperatures ---------------------------------------------------------------

# A logit over such a temperature is near a power of two from 2^54 to 2^62,
# where doubles are whole numbers apart and rounding by addition is coarser still.
TINY = [(5.933965826196662e-18, 18.966964721679688), (6.960958119566468e-18, 5.561732769012451),
        (1.6533624045163976e-18, 21.140241622924805), (2.3351737171929274e-17, 18.65730857849121),
        (2.107113983893586e-18, 13.470561027526855), (1.1937834601465037e-15, 14.591938972473145), (1e-12, 20.0), (1e-25, 3.0)]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n", [500, 9000])
def test_sample_ties_at_tiny_temperatures(n, sign):
    """Only equal largest logits have weight: top-p, top-k and min-p count them."""
    rng = np.random.default_rng(n)
    xs, rows, us = [], [], []
    for temperature, top in TINY:
        for opt in [(0, 0.5, 0.0), (0, 0.97, 0.0), (n // 2, 1.0, 0.0), (n - 1, 0.3, 0.5), (0, 1.0, 0.9)]:
            for u in (0.0, 0.4, 0.9, 1.0):
                v = (sign * top - 5.0 - 5.0 * rng.random(n)).astype(np.float32)
                v[rng.choice(n, 100, replace=False)] = np.float32(sign * top)
                xs.append(v)
                rows.append((temperature,) + opt)
                us.append(u)
    compare_samples(xs, rows, us)


# ---- batches that begin behind the first row -------------------------------------------

@pytest.mark.parametrize("many", [0, 300])
@pytest.mark.parametrize("first", [[], [(0, 30)]])
def test_rows_before_the_first_sequence(first, many):
    """A part of a larger batch: the first start is not 0. The rows before it
    are left as they were, and nothing is wrong with the batch."""
    heads, kv, dim, skip = 4, 2, 64, 5
    seqs = first + [(3, 40), (0, 9), (1, 700), (70, 90)] + [(1, 1 + i % 50) for i in range(many)]
    for shared in (0, 32):
        b, q, out, opts = attn_case([(skip, skip)] + seqs, heads, kv, dim, 16, rlh.F16, seed=many + shared, shared=shared)
        desc = b.desc()
        part = rlh.Seqs(desc.n_seq - 1, desc.n_rows, desc.max_q, desc.max_kv, desc.table_stride, b.q_start[1:].data_ptr(),
                        b.kv_len[1:].data_ptr(), b.table[1:].data_ptr())
        keep = out[:skip].clone()
        b.desc = lambda: part
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        run_attn(b, q, out, heads, status=st, **opts)
        torch.cuda.synchronize()
        assert int(st) == 0 and torch.equal(out[:skip], keep)
        whole = out.clone()
        b.desc = lambda: desc
        run_attn(b, q, whole, heads, **opts)
        torch.cuda.synchronize()
        check_attn(b, q, whole, heads, opts)
        out[:skip] = whole[:skip]
        check_attn(b, q, out, heads, opts)
        if shared:
            continue  # (some of the new rows are in the shared pages, which no sequence owns)
        b.desc = lambda: part
        x = append_inputs(b, heads, rlh.F32, 3)
        q_out = torch.full((b.n_rows, heads * dim), 7.0, dtype=torch.float16, device="cuda")
        run_append(b, x, rlh.F32, heads, q_out, None, None, None, 1.0, 0, False, st)
        torch.cuda.synchronize()
        assert int(st) == 0
        assert torch.all(q_out[:skip] == 7.0) and torch.equal(q_out[skip:], x[skip:, :heads * dim].half())
