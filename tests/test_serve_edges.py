"""Ends of the ranges that the batched serving operators accept, without a GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import rlh

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def plan_shim(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan") / "libpaged_plan_shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-o", str(out),
                    os.path.join(HERE, "paged_plan_shim.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    lib.shim_items.restype = ctypes.c_uint64
    return lib


def items(shim, steps, times, goal):
    steps, times = np.array(steps, np.uint32), np.array(times, np.uint32)
    per = ctypes.c_uint32()
    n = shim.shim_items(steps.ctypes.data_as(ctypes.c_void_p), times.ctypes.data_as(ctypes.c_void_p),
                        ctypes.c_uint32(len(steps)), ctypes.c_uint32(goal), ctypes.byref(per))
    return n, per.value


@pytest.mark.parametrize("goal", [1, 96, 768])
def test_items_fit_their_list(plan_shim, goal):
    """A list has room for `goal` items and one for each sequence, also where
    the steps of all pass 32 bits (512 sequences of 2^30 positions have 2^32:
    kept in 32 bits, their sum is 0, and more items are named than there is
    workspace for)."""
    most = (1 << 23) + 1  # 2^30 positions, 128 a step, begun inside one
    assert 65535 * most > 1 << 32
    cases = [([most], [512]), ([1 << 23], [512]), ([most], [65535]), ([most, 1], [600, 60000]), ([1], [65535]), ([1], [1])]
    rng = np.random.default_rng(goal)
    for _ in range(300):
        k = int(rng.integers(1, 6))
        cases.append((np.exp(rng.uniform(0, np.log(most), k)).astype(np.int64), rng.integers(1, 65535 // k, k)))
    for steps, times in cases:
        n, per = items(plan_shim, steps, times, goal)
        assert 1 <= per <= 1 << 24 and int(np.sum(times)) <= n <= int(np.sum(times)) + goal, (steps, times, n, per)


# ---- one workspace for all batches within limits ------------------------------------

A = 1 << 40  # spacing of addresses that are never read


def attention_args(heads, kv, dim, n_seq, n_rows, max_q, max_kv, shared, page=64):
    pool = rlh.KvPages(rlh.F16, kv, dim, page, 16, A, 2 * A)
    seqs = rlh.Seqs(n_seq, n_rows, max_q, max_kv, -(-max_kv // page), 3 * A, 4 * A, 5 * A)
    att = rlh.AttnArgs(heads, 0, 6 * A, 8 * A, heads * dim, heads * dim, 0.1, 0.0, None, None, 10 * A if shared else None,
                       shared)
    return pool, seqs, att


def log_int(rng, lo, hi):
    return int(np.exp(rng.uniform(np.log(lo), np.log(hi + 1))))


@pytest.mark.parametrize("heads,kv", [(64, 8), (16, 8), (8, 8), (12, 1), (40, 2), (28, 4), (128, 128), (512, 512)])
def test_a_workspace_serves_every_smaller_batch(heads, kv):
    """The size for some limits is accepted (as the checks before the device
    go) by every batch within them, and does not fall as limits rise."""
    rng = np.random.default_rng(heads)
    lib = rlh.load()
    for _ in range(60):
        most_q = log_int(rng, 1, 4096)
        n_seq = log_int(rng, 1, 600)
        n_rows = most_q + log_int(rng, 1, 6000) - 1
        max_kv = max(most_q, log_int(rng, 1, 60000))
        shared = 64 * log_int(rng, 1, 400) if rng.random() < 0.4 else 0
        limits = attention_args(heads, kv, 128, n_seq, n_rows, most_q, max_kv, shared)
        size = lib.rlh_paged_attn_workspace(*limits)
        for _ in range(40):
            rows = log_int(rng, 1, n_rows)
            q = min(rows, log_int(rng, 1, most_q))
            less = attention_args(heads, kv, 128, log_int(rng, 1, n_seq), rows, q, max(q, log_int(rng, 1, max_kv)),
                                  64 * int(rng.integers(0, shared // 64 + 1)))
            rc = lib.rlh_paged_attn(*less, 16 * A, size, None, None)
            assert rc in (rlh.RLH_EDEVICE, rlh.RLH_EINVAL), rc
            assert not lib.rlh_last_error().startswith(b"workspace"), (lib.rlh_last_error(), size)
            assert lib.rlh_paged_attn_workspace(*less) <= size


def test_workspace_of_a_server():
    """A prompt chunk's limits hold a token's and a short chunk's calls, and stay small."""
    lib = rlh.load()
    size = lib.rlh_paged_attn_workspace(*attention_args(64, 8, 128, 64, 4096, 4096, 40000, 0))
    assert 0 < size < 64 << 20
    for rows in (1, 100, 256, 300, 512, 2048, 4096):
        assert lib.rlh_paged_attn(*attention_args(64, 8, 128, 1, rows, rows, 40000, 0), 16 * A, size, None, None) != rlh.RLH_OK
        assert not lib.rlh_last_error().startswith(b"workspace")


# ---- what a call writes overlaps nothing else of it ----------------------------------

B = 1 << 20
D, HEADS, KV, ROWS, SEQS = 128, 4, 2, 6, 3
PLACES = dict(k_pages=1 * B, v_pages=2 * B, q_start=3 * B, kv_len=4 * B, table=5 * B, q=6 * B, k=7 * B, v=8 * B, q_norm=9 * B,
              k_norm=10 * B, freqs=11 * B, out=12 * B, slopes=13 * B, prefix_len=14 * B, shared_table=15 * B, status=16 * B,
              workspace=17 * B)
# bytes of each: 8 pages of 16 positions, rows of 640 values in all of which q takes 512
SIZE = dict(k_pages=8 * KV * 16 * D * 2, v_pages=8 * KV * 16 * D * 2, q_start=4 * (SEQS + 1), kv_len=4 * SEQS,
            table=4 * (2 * 6 + 4), q_norm=4 * D, k_norm=4 * D, freqs=8 * 64, slopes=4 * HEADS, prefix_len=4 * SEQS,
            shared_table=4, status=4)
STRIDE = 640


def call(op, **moved):
    at = {**PLACES, **moved}
    kv = rlh.KvPages(rlh.F16, KV, D, 16, 8, at["k_pages"], at["v_pages"])
    # rows of 6 page ids, of which 4 are used
    seqs = rlh.Seqs(SEQS, ROWS, 2, 60, 6, at["q_start"], at["kv_len"], at["table"])
    lib = rlh.load()
    if op == "append":
        args = rlh.AppendArgs(rlh.F16, HEADS, at["q"], at["k"], at["v"], STRIDE, STRIDE, STRIDE, at["q_norm"], at["k_norm"],
                              1e-6, 1.0, at["freqs"], 128, 0, at["out"], STRIDE)
        rc = lib.rlh_paged_append(kv, seqs, args, at["status"], None)
    else:
        args = rlh.AttnArgs(HEADS, 0, at["q"], at["out"], STRIDE, STRIDE, 0.1, 0.0, at["slopes"], at["prefix_len"],
                            at["shared_table"], 16)
        rc = lib.rlh_paged_attn(kv, seqs, args, at["workspace"], 1 << 40, at["status"], None)
    return rc, lib.rlh_last_error().decode()


READ = {"append": ["q_start", "kv_len", "table", "q_norm", "k_norm", "freqs"],
        "attn": ["q_start", "kv_len", "table", "slopes", "prefix_len", "shared_table"]}
WRITTEN = {"append": ["out", "k_pages", "v_pages"], "attn": ["out", "workspace"]}


@pytest.mark.parametrize("op", ["append", "attn"])
def test_written_memory_is_apart_from_the_arrays(op):
    name = {"out": "q_out" if op == "append" else "out", "k_pages": "the pool", "v_pages": "the pool", "workspace": "workspace"}
    assert "overlap" not in call(op)[1]
    for w in WRITTEN[op]:
        start = PLACES[w]
        for r in READ[op] + ["status"]:
            # its last bytes are the area's first, its first ones lie in a row
            unit = 16 if r.endswith("norm") else 8 if r == "freqs" else 4  # (as it has to be aligned)
            for place in (start - SIZE[r] + unit, start + 2 * STRIDE * 2 + 1008):
                rc, said = call(op, **{r: place})
                assert rc == rlh.RLH_EINVAL and said == "%s overlaps %s" % (name[w], r), (w, r, said)
    for r in READ[op] + ["q"]:
        rc, said = call(op, status=PLACES[r] + (0 if r == "q" else SIZE[r] - 4))
        assert rc == rlh.RLH_EINVAL and said == "status overlaps " + r, (r, said)
    for r in ("k_pages", "v_pages"):
        rc, said = call(op, status=PLACES[r] + SIZE[r] - 4)
        assert rc == rlh.RLH_EINVAL and "overlap" in said and "status" in said, (r, said)


@pytest.mark.parametrize("op", ["append", "attn"])
def test_memory_between_rows_is_free(op):
    """Arrays in the gap behind each output row, a status word behind a row of
    q or of the table: nothing overlaps."""
    gap = PLACES["out"] + 512 * 2
    for r in READ[op] + ["status"]:
        if SIZE[r] > 256:
            continue
        rc, said = call(op, **{r: gap + STRIDE * 2})
        assert "overlap" not in said, (r, said)
    assert "overlap" not in call(op, status=PLACES["q"] + 512 * 2)[1]
    assert "overlap" not in call(op, status=PLACES["table"] + 4 * 4)[1]
    assert "overlaps" in call(op, status=PLACES["table"] + 6 * 4)[1]
    assert "overlaps" in call(op, status=PLACES["table"] + (2 * 6 + 3) * 4)[1]
    assert "overlap" not in call(op, status=PLACES["table"] + (2 * 6 + 4) * 4)[1]
