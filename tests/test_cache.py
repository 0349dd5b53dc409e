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
        assert share >= 3 and share * n_blocks >= at
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


# ---- refusals ------------------------------------------------------------------------
# Addresses that are never read: every check below comes before the device.

OPS = ["append_at", "attn_lse", "tree_masks", "tree_attn", "tree_accept", "paged_move", "paged_mass", "evict_select"]
NODES = [f for f in BATCH if f[0] == "seqs" and f[1] in ("n_seq", "n_rows", "max_q", "q_start", "kv_len")]
CACHED = [f for f in BATCH if (f[0] == "kv" and f[2] != 3) or f[1] in ("n_seq", "kv_len", "table", "table_stride") or f[1:3] == ("max_kv", 65)]  # (no query heads: any n_head_kv)
SCORES = [("att", "n_head", 3, rlh.RLH_EINVAL), ("att", "q", 0, rlh.RLH_EINVAL), ("att", "q_stride", 513, rlh.RLH_EINVAL),
          ("att", "scale", float("inf"), rlh.RLH_EINVAL), ("att", "scale", 3e38, rlh.RLH_EINVAL),
          ("att", "softcap", -1.0, rlh.RLH_EINVAL), ("att", "slopes", A + 2, rlh.RLH_EINVAL),
          ("att", "prefix_len", A + 1, rlh.RLH_EINVAL), ("att", "shared_len", 8, rlh.RLH_EINVAL),
          ("att", "shared_len", 1 << 30, rlh.RLH_EUNSUP)]
OUT = [("att", "out", 0, rlh.RLH_EINVAL), ("att", "out", 6 * A + 512, rlh.RLH_EINVAL), ("att", "out_stride", 500, rlh.RLH_EINVAL),
       ("att", "shared_len", 16, rlh.RLH_EINVAL)]
REFUSED = {
    "append_at": test_serve.APPEND + [("", "positions", 0, rlh.RLH_EINVAL), ("", "positions", 13 * A + 2, rlh.RLH_EINVAL)],
    "attn_lse": test_serve.ATTN + [("", "lse", 0, rlh.RLH_EINVAL), ("", "lse", 14 * A + 2, rlh.RLH_EINVAL),
                                   ("", "workspace", 16 * A + 8, rlh.RLH_EINVAL)],
    "tree_masks": NODES + [("", "parents", 0, rlh.RLH_EINVAL), ("", "parents", A + 2, rlh.RLH_EINVAL),
                           ("", "masks", 0, rlh.RLH_EINVAL), ("", "masks", 15 * A + 4, rlh.RLH_EINVAL),
                           ("", "words", 0, rlh.RLH_EINVAL), ("", "words", 1 << 31, rlh.RLH_EUNSUP),
                           ("", "base", A + 1, rlh.RLH_EINVAL), ("", "positions", A + 2, rlh.RLH_EINVAL),
                           ("", "status", A + 2, rlh.RLH_EINVAL)],
    "tree_attn": BATCH + SCORES + OUT + [("att", "slopes", A, rlh.RLH_EUNSUP), ("att", "prefix_len", A, rlh.RLH_EUNSUP),
                                         ("", "masks", 0, rlh.RLH_EINVAL), ("", "masks", 15 * A + 4, rlh.RLH_EINVAL),
                                         ("", "words", 0, rlh.RLH_EINVAL), ("", "words", 1 << 31, rlh.RLH_EUNSUP),
                                         ("", "lse", 14 * A + 2, rlh.RLH_EINVAL), ("", "status", A + 2, rlh.RLH_EINVAL)],
    "tree_accept": NODES + [("acc", f, 0, rlh.RLH_EINVAL) for f in ("parents", "tokens", "sampled", "path", "count", "next",
                                                                    "new_len")] +
                   [("acc", "path", 20 * A + 1, rlh.RLH_EINVAL), ("acc", "path_stride", 4, rlh.RLH_EINVAL),
                    ("", "status", A + 2, rlh.RLH_EINVAL)],
    "paged_move": CACHED + [("mov", "index", 0, rlh.RLH_EINVAL), ("mov", "index", A + 2, rlh.RLH_EINVAL),
                            ("mov", "count", 0, rlh.RLH_EINVAL), ("mov", "max_count", 21, rlh.RLH_EINVAL),
                            ("mov", "mass", 0, rlh.RLH_EINVAL), ("mov", "mass_out", 0, rlh.RLH_EINVAL),
                            ("mov", "base", A + 2, rlh.RLH_EINVAL), ("mov", "mass_out", 25 * A + 64, rlh.RLH_EINVAL),
                            ("", "status", A + 2, rlh.RLH_EINVAL)],
    "paged_mass": BATCH + SCORES + [("", "lse", 0, rlh.RLH_EINVAL), ("", "lse", A + 2, rlh.RLH_EINVAL), ("", "mass", 0, rlh.RLH_EINVAL),
                                    ("", "mass", 25 * A + 8, rlh.RLH_EINVAL), ("", "decay", -0.5, rlh.RLH_EINVAL),
                                    ("", "decay", float("inf"), rlh.RLH_EINVAL), ("", "decay", float("nan"), rlh.RLH_EINVAL),
                                    ("", "status", A + 2, rlh.RLH_EINVAL)],
    "evict_select": CACHED + [("evi", "mass", 0, rlh.RLH_EINVAL), ("evi", "mass", A + 2, rlh.RLH_EINVAL), ("evi", "keep", 0, rlh.RLH_EINVAL),
                              ("evi", "count", 0, rlh.RLH_EINVAL), ("evi", "budget", 0, rlh.RLH_EINVAL),
                              ("evi", "first_kept", 15, rlh.RLH_EINVAL), ("evi", "last_kept", 0xffffffff, rlh.RLH_EINVAL),
                              ("evi", "keep_stride", 19, rlh.RLH_EINVAL), ("", "status", A + 2, rlh.RLH_EINVAL)],
}


def good():
    args = test_serve.good()
    args["acc"] = dict(parents=17 * A, tokens=18 * A, sampled=19 * A, path=20 * A, path_stride=5, count=21 * A, next=22 * A,
                       new_len=23 * A)
    args["mov"] = dict(index=24 * A, index_stride=20, per_head=1, count=21 * A, max_count=20, base=0, mass=25 * A, mass_out=26 * A)
    args["evi"] = dict(mass=25 * A, budget=20, first_kept=4, last_kept=6, keep_stride=20, keep=27 * A, count=21 * A)
    args[""] = dict(positions=13 * A, lse=14 * A, masks=15 * A, words=1, parents=17 * A, base=28 * A, workspace=16 * A, status=0,
                    mass=25 * A, decay=0.5)
    return args


def call(op, args):
    lib = rlh.load()
    kv, seqs, app, att = test_serve.structs(args)
    x = args[""]
    st = x["status"] or None
    if op == "append_at":
        rc = lib.rlh_paged_append_at(kv, seqs, app, x["positions"], st, None)
    elif op == "attn_lse":
        rc = lib.rlh_paged_attn_lse(kv, seqs, att, x["lse"], x["workspace"], 1 << 40, st, None)
    elif op == "tree_masks":
        rc = lib.rlh_tree_masks(seqs, x["parents"], x["base"], x["masks"], x["words"], x["positions"], st, None)
    elif op == "tree_attn":
        rc = lib.rlh_tree_attn(kv, seqs, att, x["masks"], x["words"], x["lse"], x["workspace"], 1 << 40, st, None)
    elif op == "tree_accept":
        rc = lib.rlh_tree_accept(seqs, rlh.AcceptArgs(**args["acc"]), st, None)
    elif op == "paged_move":
        rc = lib.rlh_paged_move(kv, seqs, rlh.MoveArgs(**args["mov"]), st, None)
    elif op == "paged_mass":
        rc = lib.rlh_paged_mass(kv, seqs, att, x["lse"], x["decay"], x["mass"], st, None)
    else:
        rc = lib.rlh_evict_select(kv, seqs, rlh.EvictArgs(**args["evi"]), st, None)
    return rc, lib.rlh_last_error().decode()


def _has_gpu():
    import torch

    return torch.cuda.device_count() > 0


@pytest.mark.parametrize("op", OPS)
def test_refusals(op):
    for part, field, value, code in REFUSED[op]:
        args = good()
        args[part][field] = value
        rc, said = call(op, args)
        assert rc == code and said, (part, field, value, rc, said)


@pytest.mark.parametrize("op", OPS)
def test_missing_structs(op):
    lib, f = rlh.load(), {"append_at": "rlh_paged_append_at", "attn_lse": "rlh_paged_attn_lse"}.get(op, "rlh_" + op)
    f = getattr(lib, f)
    args = good()
    kv, seqs, app, att = test_serve.structs(args)
    own = {"append_at": app, "attn_lse": att, "tree_attn": att, "paged_mass": att, "tree_accept": rlh.AcceptArgs(**args["acc"]),
           "paged_move": rlh.MoveArgs(**args["mov"]), "evict_select": rlh.EvictArgs(**args["evi"])}
    lead = [seqs] if op in ("tree_masks", "tree_accept") else [kv, seqs]
    lead += [own[op]] if op in own else []
    rest = [0.5 if t is ctypes.c_float else 1 if t in (U32, U64) else 16 * A for t in f.argtypes[len(lead):]]
    rest[-2:] = [None, None]
    for i in range(len(lead)):
        assert f(*(lead[:i] + [None] + lead[i + 1:]), *rest) == rlh.RLH_EINVAL


@pytest.mark.skipif(_has_gpu(), reason="checks the no-GPU error path")
@pytest.mark.parametrize("op", OPS)
def test_what_is_accepted_needs_a_device(op):
    rc, said = call(op, good())
    assert rc == rlh.RLH_EDEVICE and "no HIP device" in said, said


@pytest.mark.parametrize("op", OPS)
def test_empty_batches_do_nothing(op):
    args = good()
    args["seqs"]["n_seq"] = 0
    assert call(op, args)[0] == rlh.RLH_OK
    args = good()
    args["seqs"]["n_rows"] = 0
    if op in ("tree_accept", "paged_move", "evict_select"):  # these have work without rows
        args["seqs"].update(max_q=0, q_start=3 * A if op == "tree_accept" else 0)
        if op == "tree_accept":
            args["acc"].update(parents=0, tokens=0, sampled=0, path=0)
        assert call(op, args)[0] in (rlh.RLH_EDEVICE, rlh.RLH_EINVAL) and "null" not in call(op, args)[1]
    else:
        args[""].update(lse=0 if op == "attn_lse" else 14 * A, masks=0 if op == "tree_attn" else 15 * A)
        assert call(op, args)[0] == rlh.RLH_OK
    args = good()
    args["mov"]["max_count"] = 0
    if op == "paged_move":
        assert call(op, args)[0] == rlh.RLH_OK


# what a call writes and reads: (part, field) and bytes
POOL = 8 * 2 * 16 * 128 * 2
READS = {"q_start": ("seqs", "q_start", 12), "kv_len": ("seqs", "kv_len", 8), "table": ("seqs", "table", 32),
         "positions": ("", "positions", 24), "masks": ("", "masks", 48), "parents": ("", "parents", 24), "base": ("", "base", 8),
         "lse": ("", "lse", 96), "a.parents": ("acc", "parents", 24), "tokens": ("acc", "tokens", 24),
         "sampled": ("acc", "sampled", 24), "index": ("mov", "index", 320), "m.count": ("mov", "count", 8),
         "m.base": ("mov", "base", 8), "mass": ("", "mass", 1024), "e.mass": ("evi", "mass", 1024), "q": ("att", "q", 6144),
         "k": ("kv", "k", POOL), "v": ("kv", "v", POOL)}
APART = {
    "append_at": [(("app", "q_out", 6144), ["positions"]), (("kv", "k", POOL), ["positions"])],
    "attn_lse": [(("", "lse", 96), ["q_start", "kv_len", "table", "q", "k", "v"])],
    "tree_masks": [(("", "masks", 48), ["q_start", "kv_len", "parents", "base", "positions"]),
                   (("", "positions", 24), ["q_start", "kv_len", "parents", "base"])],
    "tree_attn": [(("att", "out", 6144), ["masks"]), (("", "lse", 96), ["q_start", "kv_len", "table", "masks", "q", "k", "v"])],
    "tree_accept": [(("acc", f, n), ["q_start", "kv_len", "a.parents", "tokens", "sampled"])
                    for f, n in (("path", 40), ("count", 8), ("next", 8), ("new_len", 8))],
    "paged_move": [(("kv", f, POOL), ["kv_len", "table", "index", "m.count", "m.base"]) for f in ("k", "v")] +
                  [(("mov", "mass_out", 1024), ["kv_len", "table", "index", "m.count", "m.base", "k", "v"])],
    "paged_mass": [(("", "mass", 1024), ["q_start", "kv_len", "table", "q", "lse", "k", "v"])],
    "evict_select": [(("evi", "keep", 320), ["kv_len", "table", "e.mass"]), (("evi", "count", 8), ["kv_len", "table", "e.mass"])],
}


@pytest.mark.parametrize("op", OPS)
def test_written_memory_is_apart(op):
    for (part, field, size), names in APART[op]:
        for name in names + ["status"]:
            for at in (0, 1):  # its first bytes are the area's last ones, its last ones the area's first
                args = good()
                start = args[part][field]
                p2, f2, n2 = READS[name] if name != "status" else ("", "status", 4)
                unit = 16 if name in ("q", "k", "v", "mass") else 8 if name == "masks" else 4
                place = start + size - unit if at == 0 else start - n2 + unit
                if place % unit or (field in ("masks", "mass", "k", "v", "q_out", "out") and n2 % unit):
                    continue
                args[p2][f2] = place
                rc, said = call(op, args)
                assert rc == rlh.RLH_EINVAL and "overlap" in said, (field, name, at, said)


@pytest.mark.parametrize("heads,kv", [(64, 8), (16, 8), (12, 1), (40, 2), (28, 4), (128, 128), (512, 512), (24, 1)])
def test_a_tree_workspace_serves_every_smaller_batch(heads, kv):
    """As of rlh_paged_attn: the size for some limits is enough for every batch within them."""
    from test_serve_edges import A as far
    from test_serve_edges import attention_args, log_int

    rng = np.random.default_rng(heads)
    lib = rlh.load()
    for _ in range(60):
        most_q, n_seq, shared = log_int(rng, 1, 700), log_int(rng, 1, 600), 64 * log_int(rng, 1, 100) if rng.random() < 0.4 else 0
        n_rows, max_kv = most_q + log_int(rng, 1, 6000) - 1, max(most_q, log_int(rng, 1, 60000))
        size = lib.rlh_tree_attn_workspace(*attention_args(heads, kv, 128, n_seq, n_rows, most_q, max_kv, shared))
        for _ in range(40):
            rows = log_int(rng, 1, n_rows)
            q = min(rows, log_int(rng, 1, most_q))
            less = attention_args(heads, kv, 128, log_int(rng, 1, n_seq), rows, q, max(q, log_int(rng, 1, max_kv)),
                                  64 * int(rng.integers(0, shared // 64 + 1)))
            rc = lib.rlh_tree_attn(*less, 12 * far, 16, None, 16 * far, size, None, None)
            assert rc in (rlh.RLH_EDEVICE, rlh.RLH_EINVAL), rc
            assert not lib.rlh_last_error().startswith(b"workspace"), (lib.rlh_last_error(), size)
            assert lib.rlh_tree_attn_workspace(*less) <= size


def test_tree_workspace_of_a_server():
    """64 sequences of up to 63 nodes at 40000 positions: parts of 256 blocks, two each."""
    from test_serve_edges import A as far
    from test_serve_edges import attention_args

    lib = rlh.load()
    args = attention_args(64, 8, 128, 64, 4032, 63, 40000, 0)
    size = lib.rlh_tree_attn_workspace(*args)
    assert 0 < size < 72 << 20
    lib.rlh_tree_attn(*args, 12 * far, 1, None, 16 * far, size // 2, None, None)
    assert lib.rlh_last_error().startswith(b"workspace")
