"""The operators that edit a paged cache (include/rlh_cache.h) without a GPU:
the header and its bindings, refusals, overlaps, workspace bounds, and the index
rules that the kernels share with the host (tests/tree_index_shim.cpp)."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import rlh
import test_serve
from test_serve import A, BATCH, C_TO_CTYPES, rust_type

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
U32, U64, I32 = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int32


# ---- header and bindings ----------------------------------------------------------

STRUCTS = {"rlh_accept_args": rlh.AcceptArgs, "rlh_move_args": rlh.MoveArgs, "rlh_evict_args": rlh.EvictArgs}


@pytest.fixture
def header(monkeypatch):
    text = open(os.path.join(ROOT, "include", "rlh_cache.h")).read()
    text = re.sub(r"#.*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))
    monkeypatch.setattr(test_serve, "header", lambda: text)
    return text


def rust_block():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    blocks = [b for b in re.findall(r"```rs\n(.*?)```", text, flags=re.S) if "RlhMoveArgs" in b]
    assert len(blocks) == 1
    return blocks[0]


def test_library_exports_the_header(header):
    lib = ctypes.CDLL(rlh.LIB_PATH)
    names = test_serve.header_functions()
    assert len(names) == 9
    assert not [n for n in names if not hasattr(lib, n)]


def test_structs_match_their_bindings(header):
    rust, structs = rust_block(), test_serve.header_structs()
    assert sorted(structs) == sorted(STRUCTS)
    for name, fields in structs.items():
        py = STRUCTS[name]._fields_
        assert [n for n, _ in py] == [n for _, n in fields], name
        for (_, got), (ctype, field) in zip(py, fields):
            assert got is (ctypes.c_void_p if "*" in ctype else C_TO_CTYPES[ctype]), (name, field)
        camel = "".join(p.capitalize() for p in name.split("_"))
        body = re.search(r"pub struct %s \{(.*?)\}" % camel, rust, flags=re.S).group(1)
        got = [tuple(x.strip() for x in f.replace("pub ", "").split(":")) for f in body.split(",") if f.strip()]
        assert got == [(n, rust_type(t)) for t, n in fields], name


def test_functions_match_their_bindings(header):
    got = {}
    for m in re.finditer(r"pub fn (rlh_\w+)\((.*?)\) -> (\w+);", rust_block(), flags=re.S):
        got[m.group(1)] = (m.group(3), [tuple(x.strip() for x in a.split(":")) for a in " ".join(m.group(2).split()).split(",")])
    functions = test_serve.header_functions()
    want = {n: (test_serve.C_TO_RUST[r], [(p, rust_type(t)) for t, p in ps]) for n, (r, ps) in functions.items()}
    assert got == want
    lib = rlh.load()
    for name, (ret, params) in functions.items():
        f = getattr(lib, name)
        assert f.restype is (U64 if ret == "uint64_t" else I32), name
        for got, (ctype, field) in zip(f.argtypes, params):
            if "*" in ctype:
                assert got is ctypes.c_void_p or issubclass(got, ctypes._Pointer), (name, field)
            else:
                assert got is C_TO_CTYPES[ctype], (name, field)
        assert len(f.argtypes) == len(params)


# ---- index rules ----------------------------------------------------------------------

@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = tmp_path_factory.mktemp("tree") / "libtree_index_shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-o", str(out),
                    os.path.join(HERE, "tree_index_shim.cpp")], check=True)
    lib = ctypes.CDLL(str(out))
    lib.shim_line_units.restype = lib.shim_line_share.restype = U64
    return lib


def ptr(x):
    return x.ctypes.data_as(ctypes.c_void_p)


def test_what_drafted_rows_see(shim):
    rng = np.random.default_rng(1)
    for _ in range(2000):
        q = int(rng.choice([1, 2, 63, 64, 65, 127, 128, int(rng.integers(1, 200))]))
        words = (q + 63) // 64 + int(rng.integers(0, 2))
        first = int(rng.choice([0, 1, 15, int(rng.integers(0, 300))]))
        window = int(rng.choice([0, 0, 1, 3, q, int(rng.integers(1, 400)), 0x80000000, 0xffffffff]))
        bits = rng.random((words, 64)) < rng.choice([0.0, 0.1, 0.9, 1.0])
        mask = np.packbits(bits.reshape(-1), bitorder="little").view(np.uint64).copy()
        see = bits.reshape(-1)[:q]
        n = first + q
        sees = np.zeros(n, np.uint8)
        got = shim.shim_tree_sees(ptr(mask), U32(words), U32(q), I32(first), U32(window), I32(-int(rng.integers(0, 64))), ptr(sees),
                                  U32(n))
        assert got == see.sum()
        j = np.arange(first)
        want = np.concatenate([j >= first + see.sum() - window if window else j >= 0, see])
        assert np.array_equal(sees.astype(bool), want)


def test_a_line_of_tiles_is_divided_once(shim):
    """Every step of every tile belongs to one block; what a block leaves of a
    tile lies in a place of its own, which is where the parts are looked for."""
    rng = np.random.default_rng(2)
    out, blocks, slots = (U32 * 4 * 4096)(), (U32 * 2)(), (U32 * 4096)()
    for _ in range(400):
        n_seq = int(rng.integers(1, 12))
        rows = [int(rng.choice([0, 1, 16, 128, 129, 256, 257, int(np.exp(rng.uniform(0, 7.5)))])) for _ in range(n_seq)]
        steps = [int(np.exp(rng.uniform(0, rng.choice([1.0, 4.0, 7.0])))) for _ in range(n_seq)]
        n_blocks = int(rng.choice([1, 2, 6, 32, 85, 256]))
        first, at = [], 0
        for r, st in zip(rows, steps):
            first.append(at)
            at += shim.shim_line_units(U32(r), U32(st))
        if at == 0:
            continue
        share = shim.shim_line_share(U64(at), U32(n_blocks))
        assert share >= 12 and share * n_blocks >= at
        used = {}
        done = [np.zeros(((r + 255) // 256, st), int) for r, st in zip(rows, steps)]
        whole = set()
        for s in range(n_seq):
            if rows[s] == 0:
                continue
            for b in range(n_blocks):
                for i in range(shim.shim_line_block(U64(first[s]), U32(rows[s]), U32(steps[s]), U64(share), U32(b), out)):
                    k, st0, st1, slot = out[i]
                    done[s][k, st0:st1] += 1
                    if st0 >= st1:
                        continue
                    if (st0, st1) == (0, steps[s]):
                        whole.add((s, k))
                    else:
                        assert slot < 2 * n_blocks and slot not in used, (s, k, b)
                        used[slot] = (s, k, b)
            assert np.all(done[s] == 1)
            for k in range((rows[s] + 255) // 256):
                shim.shim_line_parts(U64(first[s]), U32(rows[s]), U32(steps[s]), U64(share), U32(k), blocks, slots)
                assert blocks[0] <= blocks[1] < n_blocks
                assert ((s, k) in whole) == (blocks[0] == blocks[1])
                if blocks[0] != blocks[1]:
                    for b in range(blocks[0], blocks[1] + 1):
                        assert used.pop(slots[b - blocks[0]]) == (s, k, b)
        assert not used


def test_a_line_past_32_bits(shim):
    """2^30 positions of 2^25 rows."""
    rows, steps = 1 << 25, (1 << 24) + 1
    units = shim.shim_line_units(U32(rows), U32(steps))
    assert units == (1 << 17) * 3 * (steps + 2)
    share = shim.shim_line_share(U64(units), U32(32))
    out, n = (U32 * 4 * 8192)(), 0
    for b in (0, 31):
        got = shim.shim_line_block(U64(0), U32(rows), U32(steps), U64(share), U32(b), out)
        assert out[0][0] == b * 4096 and got == 4096 and [out[got - 1][i] for i in range(3)] == [b * 4096 + 4095, 0, steps]
