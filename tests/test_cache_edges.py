"""The operators that edit a paged cache (include/rlh_cache.h) without a GPU:
windows shorter than what drafted rows see of each other."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import rlh
from test_cache import ROOT, I32, U32, U64, _has_gpu, call, good, ptr
from test_serve_edges import A as far
from test_serve_edges import attention_args, log_int

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = tmp_path_factory.mktemp("window") / "libtree_window_shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-o", str(out),
                    os.path.join(HERE, "tree_window_shim.cpp")], check=True)
    return ctypes.CDLL(str(out))


def row_sees(shim, bits, q, first, window, start=0):
    mask = np.packbits(bits.reshape(-1), bitorder="little").view(np.uint64).copy()
    sees, left = np.zeros(first + q, np.uint8), np.zeros_like(mask)
    shim.shim_row_sees(ptr(mask), U32(len(mask)), U32(q), I32(first), U32(window), ptr(left), I32(start), ptr(sees), U32(first + q))
    return sees.astype(bool)


def test_a_window_that_bounds_the_drafts(shim):
    """Of all that a row would see without a window, before its batch and in
    it, the last `window`."""
    rng = np.random.default_rng(5)
    cut = 0
    for _ in range(3000):
        q = int(rng.choice([1, 2, 63, 64, 65, 127, 128, 129, int(rng.integers(1, 260))]))
        words = (q + 63) // 64 + int(rng.integers(0, 2))
        first = int(rng.choice([0, 1, 15, int(rng.integers(0, 300))]))
        window = int(rng.choice([0, 1, 2, 3, q, int(rng.integers(1, 400)), 0x7fffffff]))
        bits = rng.random((words, 64)) < rng.choice([0.0, 0.1, 0.5, 0.9, 1.0])
        see = bits.reshape(-1)[:q]
        line = np.concatenate([np.arange(first), first + np.flatnonzero(see)])
        want = np.zeros(first + q, bool)
        want[line[-window:] if window else line] = True
        assert np.array_equal(row_sees(shim, bits, q, first, window, -int(rng.integers(0, 64))), want)
        cut += bool(window) and see.sum() > window
    assert cut > 500


def test_a_chain_under_a_window_sees_what_the_attention_does(shim):
    for q, first, window in ((1, 0, 1), (5, 3, 2), (70, 10, 1), (70, 0, 64), (130, 200, 65), (200, 30, 199), (64, 64, 64), (9, 40, 20)):
        for i in range(q):
            bits = np.zeros((q + 63) // 64 * 64, bool)
            bits[:i + 1] = True
            j = np.arange(first + q)
            assert np.array_equal(row_sees(shim, bits, q, first, window), (j <= first + i) & (j > first + i - window))


def test_the_flag_of_the_window():
    text = open(os.path.join(ROOT, "include", "rlh_cache.h")).read()
    assert "#define RLH_WINDOW_DRAFTS 0x80000000u" in text and rlh.WINDOW_DRAFTS == 0x80000000


@pytest.mark.parametrize("heads,kv", [(64, 8), (16, 8), (12, 1), (24, 1)])
def test_a_tree_workspace_for_windows_serves_every_smaller_batch(heads, kv):
    """Asked for with the flag, it holds what a window of any length takes of
    smaller batches, and a batch without the flag."""
    rng = np.random.default_rng(heads)
    lib = rlh.load()
    for _ in range(40):
        most_q, n_seq, shared = log_int(rng, 1, 700), log_int(rng, 1, 600), 64 * log_int(rng, 1, 100) if rng.random() < 0.4 else 0
        n_rows, max_kv = most_q + log_int(rng, 1, 6000) - 1, max(most_q, log_int(rng, 1, 60000))

        def attention(*sizes, window):
            args = attention_args(heads, kv, 128, *sizes)
            args[2].window = window
            return args

        limits = attention(n_seq, n_rows, most_q, max_kv, shared, window=rlh.WINDOW_DRAFTS | log_int(rng, 1, 1000))
        size = lib.rlh_tree_attn_workspace(*limits)
        for _ in range(40):
            rows = log_int(rng, 1, n_rows)
            q = min(rows, log_int(rng, 1, most_q))
            less = attention(log_int(rng, 1, n_seq), rows, q, max(q, log_int(rng, 1, max_kv)), 64 * int(rng.integers(0, shared // 64 + 1)),
                             window=int(rng.choice([0, rlh.WINDOW_DRAFTS])) | log_int(rng, 1, 1000))
            rc = lib.rlh_tree_attn(*less, 12 * far, 16, None, 16 * far, size, None, None)
            assert rc in (rlh.RLH_EDEVICE, rlh.RLH_EINVAL), rc
            assert not lib.rlh_last_error().startswith(b"workspace"), (lib.rlh_last_error(), size)
            assert lib.rlh_tree_attn_workspace(*less) <= size
    # eight rows whose window cuts their masks take eight words more (256 bytes), any other eight rows none
    def needed(window):
        lib.rlh_tree_attn(*attention(1, 8, 8, 1000, 0, window=window), 12 * far, 1, None, 16 * far, 0, None, None)
        return int(lib.rlh_last_error().split(b" bytes, ")[1].split()[0])

    assert needed(rlh.WINDOW_DRAFTS | 4) == needed(4) + 256
    assert needed(rlh.WINDOW_DRAFTS | 8) == needed(rlh.WINDOW_DRAFTS) == needed(4)


@pytest.mark.skipif(_has_gpu(), reason="checks the no-GPU error path")
@pytest.mark.parametrize("stride", [0, 4])
@pytest.mark.parametrize("op", ["paged_move", "evict_select"])
def test_batches_of_empty_sequences_are_taken(op, stride):
    """max_kv 0: every sequence is empty, its count is written all the same.
    An array of no bytes overlaps nothing."""
    args = good()
    args["seqs"].update(max_kv=0, max_q=0, n_rows=0, q_start=0, table_stride=stride)
    args["evi"]["keep_stride"] = 0
    for table in (args["seqs"]["table"], args["evi"]["mass"] + 64, args["kv"]["k"] + 64):
        args["seqs"]["table"] = table
        rc, said = call(op, args)
        assert rc == rlh.RLH_EDEVICE and "no HIP device" in said, (said, table)


# ---- that the GPU tests reach what they are for -----------------------------------------

@pytest.fixture(scope="module")
def line(tmp_path_factory):
    out = tmp_path_factory.mktemp("line") / "libtree_index_shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(out), os.path.join(HERE, "tree_index_shim.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    lib.shim_line_units.restype = lib.shim_line_share.restype = U64
    return lib


def test_long_jobs_are_long(line):
    """The steps that one block takes of one tile, in the batches of
    test_gpu_cache_edges.py: more than 32, and the first job of the line too."""
    from test_gpu_cache_edges import LONG_JOBS

    out = (U32 * 4 * 4096)()
    for name, case in LONG_JOBS.items():
        group, shared, window = case["heads"] // case["kv"], case.get("shared", 0), case.get("window", 0)
        tiles = [(sum(q for q, _ in case["seqs"]) * group, shared // 64)] if shared else []
        for q, n in case["seqs"]:
            begin = max(shared, n - q - window if window else 0) // 16 * 16
            tiles.append((q * group, -(-(n - begin) // 64)))
        at, firsts = 0, []
        for rows, steps in tiles:
            firsts.append(at)
            at += line.shim_line_units(U32(rows), U32(steps))
        blocks = max(1, 256 // case["kv"])
        share = line.shim_line_share(U64(at), U32(blocks))
        jobs = []
        for first, (rows, steps) in zip(firsts, tiles):
            for block in range(blocks):
                for i in range(line.shim_line_block(U64(first), U32(rows), U32(steps), U64(share), U32(block), out)):
                    jobs.append(out[i][2] - out[i][1])
        assert jobs[0] > 36, (name, jobs)


def test_weights_go_on_from_step_to_step():
    from test_gpu_cache_edges import GOES_ON

    for name, case in GOES_ON.items():
        few = max(q for q, _ in case["seqs"]) * (case["heads"] // case["kv"]) <= 16
        steps = -(-(max(n for _, n in case["seqs"]) - case.get("shared", 0)) // 128)
        blocks = max(1, (4096 if few else 65536) // (len(case["seqs"]) * case["kv"]))
        assert steps > 2 * blocks and few == ("rows" not in name), name
