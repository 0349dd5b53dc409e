"""Ends of the ranges that the batched serving operators accept, without a GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

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
