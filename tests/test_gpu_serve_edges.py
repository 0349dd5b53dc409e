"""Ends of the ranges that the batched serving operators accept, on the GPU
against 64-bit forms."""
import numpy as np
import pytest
import torch

import rlh
import serve_ref as ref
from test_gpu_serve import run_sample

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
