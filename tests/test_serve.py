"""The batched serving operators without a GPU: the header, its Rust and
ctypes bindings, refusals, rotary frequencies, and the index rules that the
kernels share with the host (tests/paged_index_shim.cpp)."""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest

import rlh

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


# ---- header and bindings ----------------------------------------------------------

C_TO_RUST = {"int": "c_int", "uint32_t": "u32", "uint64_t": "u64", "float": "f32", "double": "f64", "void": "c_void"}
C_TO_CTYPES = {"uint32_t": ctypes.c_uint32, "uint64_t": ctypes.c_uint64, "float": ctypes.c_float,
               "double": ctypes.c_double}
STRUCTS = {"rlh_kv_pages": rlh.KvPages, "rlh_seqs": rlh.Seqs, "rlh_rope": rlh.Rope, "rlh_append_args": rlh.AppendArgs,
           "rlh_attn_args": rlh.AttnArgs, "rlh_row_sampling": rlh.RowSampling}


def header():
    text = open(os.path.join(ROOT, "include", "rlh_serve.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.sub(r"#.*", "", text)


def rust_type(ctype):
    base = [t for t in ctype.replace("*", " ").split() if t != "const"][0]
    out = C_TO_RUST.get(base) or "".join(p.capitalize() for p in base.split("_"))
    if "*" in ctype:
        out = ("*const " if ctype.split()[0] == "const" else "*mut ") + out
    return out


def header_structs():
    found = {}
    for m in re.finditer(r"typedef struct (\w+) \{(.*?)\}", header(), flags=re.S):
        fields = []
        for line in m.group(2).split(";"):
            line = " ".join(line.split())
            if not line:
                continue
            first, *more = line.split(",")
            ctype, name = re.match(r"(.*?[\s\*])(\w+)$", first).groups()
            fields += [(ctype.strip(), n.strip()) for n in [name] + more]
        found[m.group(1)] = fields
    return found


def header_functions():
    found = {}
    for m in re.finditer(r"(int|uint64_t) (rlh_\w+)\(([^)]*)\);", header()):
        params = [re.match(r"(.*?[\s\*])(\w+)$", " ".join(a.split())).groups() for a in m.group(3).split(",")]
        found[m.group(2)] = (m.group(1), [(t.strip(), n) for t, n in params])
    return found


def rust_block():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    blocks = [b for b in re.findall(r"```rust\n(.*?)```", text, flags=re.S) if "RlhKvPages" in b]
    assert len(blocks) == 1
    return blocks[0]


def test_library_exports_the_header():
    lib = ctypes.CDLL(rlh.LIB_PATH)
    names = header_functions()
    assert len(names) == 6
    assert not [n for n in names if not hasattr(lib, n)]


def test_structs_match_their_bindings():
    rust = rust_block()
    structs = header_structs()
    assert sorted(structs) == sorted(STRUCTS)
    for name, fields in structs.items():
        py = STRUCTS[name]._fields_
        assert [n for n, _ in py] == [n for _, n in fields], name
        for (_, got), (ctype, field) in zip(py, fields):
            assert got is (ctypes.c_void_p if "*" in ctype else C_TO_CTYPES[ctype]), (name, field)
        camel = "".join(p.capitalize() for p in name.split("_"))
        body = re.search(r"pub struct %s \{(.*?)\}" % camel, rust, flags=re.S).group(1)
        got = [tuple(x.strip() for x in f.replace("pub ", "").replace("r#", "").split(":")) for f in body.split(",") if f.strip()]
        assert got == [(n, rust_type(t)) for t, n in fields], name


def test_functions_match_their_binding():
    rust = rust_block()
    got = {}
    for m in re.finditer(r"pub fn (rlh_\w+)\((.*?)\) -> (\w+);", rust, flags=re.S):
        got[m.group(1)] = (m.group(3), [tuple(x.strip().replace("r#", "") for x in a.split(":"))
                                        for a in " ".join(m.group(2).split()).split(",")])
    want = {n: (C_TO_RUST[r], [(p, rust_type(t)) for t, p in ps]) for n, (r, ps) in header_functions().items()}
    assert got == want


# ---- refusals ------------------------------------------------------------------------
# Addresses that are never read: every check below comes before the device.

A = 1 << 20  # spacing of the made-up buffers


def good():
    kv = dict(type=rlh.BF16, n_head_kv=2, head_dim=128, page_size=16, n_pages=8, k=A, v=2 * A)
    seqs = dict(n_seq=2, n_rows=6, max_q=5, max_kv=60, table_stride=4, q_start=3 * A, kv_len=4 * A, table=5 * A)
    app = dict(in_type=rlh.F32, n_head=4, q=6 * A, k=7 * A, v=8 * A, q_stride=512, k_stride=256, v_stride=256,
               q_norm=9 * A, k_norm=10 * A, eps=1e-6, magnitude=1.0, freqs=11 * A, rot_dim=128, interleaved=0,
               q_out=12 * A, q_out_stride=512)
    att = dict(n_head=4, window=0, q=6 * A, out=7 * A, q_stride=512, out_stride=512, scale=0.1, softcap=0.0, slopes=0,
               prefix_len=0, shared_table=0, shared_len=0)
    return {"kv": kv, "seqs": seqs, "app": app, "att": att}


BATCH = [("kv", "type", rlh.F32, rlh.RLH_EUNSUP), ("kv", "type", 99, rlh.RLH_EUNSUP), ("kv", "head_dim", 96, rlh.RLH_EUNSUP),
         ("kv", "head_dim", 0, rlh.RLH_EUNSUP), ("kv", "page_size", 8, rlh.RLH_EUNSUP),
         ("kv", "page_size", 48, rlh.RLH_EUNSUP), ("kv", "page_size", 512, rlh.RLH_EUNSUP),
         ("kv", "n_head_kv", 3, rlh.RLH_EINVAL), ("kv", "n_head_kv", 0, rlh.RLH_EINVAL), ("kv", "n_pages", 0, rlh.RLH_EINVAL),
         ("kv", "n_pages", 1 << 31, rlh.RLH_EINVAL), ("kv", "k", 0, rlh.RLH_EINVAL), ("kv", "v", A + 16, rlh.RLH_EINVAL),
         ("kv", "k", A + 8, rlh.RLH_EINVAL), ("seqs", "n_seq", 65536, rlh.RLH_EUNSUP),
         ("seqs", "n_rows", 1 << 24, rlh.RLH_EUNSUP), ("seqs", "max_q", 0, rlh.RLH_EINVAL), ("seqs", "max_q", 7, rlh.RLH_EINVAL),
         ("seqs", "max_kv", 4, rlh.RLH_EINVAL), ("seqs", "max_kv", 65, rlh.RLH_EINVAL), ("seqs", "q_start", 0, rlh.RLH_EINVAL),
         ("seqs", "kv_len", 0, rlh.RLH_EINVAL), ("seqs", "table", 0, rlh.RLH_EINVAL), ("seqs", "table", 5 * A + 2, rlh.RLH_EINVAL),
         ("seqs", "table_stride", 1 << 26, rlh.RLH_EUNSUP)]
APPEND = BATCH + [("app", "n_head", 5, rlh.RLH_EINVAL), ("app", "n_head", 2048, rlh.RLH_EUNSUP),
                  ("app", "in_type", rlh.Q8_0, rlh.RLH_EUNSUP), ("app", "q", 0, rlh.RLH_EINVAL),
                  ("app", "k", 0, rlh.RLH_EINVAL), ("app", "v", 0, rlh.RLH_EINVAL), ("app", "q_out", 0, rlh.RLH_EINVAL),
                  ("app", "q", 6 * A + 4, rlh.RLH_EINVAL), ("app", "q_stride", 511, rlh.RLH_EINVAL),
                  ("app", "q_stride", 514, rlh.RLH_EINVAL), ("app", "k_stride", 128, rlh.RLH_EINVAL),
                  ("app", "v_stride", 1 << 33, rlh.RLH_EINVAL), ("app", "q_out_stride", 516, rlh.RLH_EINVAL),
                  ("app", "rot_dim", 8, rlh.RLH_EINVAL), ("app", "rot_dim", 144, rlh.RLH_EINVAL),
                  ("app", "freqs", 0, rlh.RLH_EINVAL), ("app", "freqs", 11 * A + 4, rlh.RLH_EINVAL),
                  ("app", "q_norm", 9 * A + 4, rlh.RLH_EINVAL), ("app", "q_out", 6 * A, rlh.RLH_EINVAL),
                  ("app", "q_out", 7 * A + 16, rlh.RLH_EINVAL)]
ATTN = BATCH + [("att", "n_head", 3, rlh.RLH_EINVAL), ("att", "q", 0, rlh.RLH_EINVAL), ("att", "out", 0, rlh.RLH_EINVAL),
                ("att", "out", 6 * A + 512, rlh.RLH_EINVAL), ("att", "out_stride", 500, rlh.RLH_EINVAL),
                ("att", "q_stride", 513, rlh.RLH_EINVAL), ("att", "scale", math.inf, rlh.RLH_EINVAL),
                ("att", "scale", math.nan, rlh.RLH_EINVAL), ("att", "softcap", -1.0, rlh.RLH_EINVAL),
                ("att", "softcap", math.inf, rlh.RLH_EINVAL), ("att", "softcap", math.nan, rlh.RLH_EINVAL),
                ("att", "slopes", A + 2, rlh.RLH_EINVAL), ("att", "prefix_len", A + 1, rlh.RLH_EINVAL),
                ("att", "shared_len", 8, rlh.RLH_EINVAL), ("att", "shared_len", 16, rlh.RLH_EINVAL),
                ("att", "shared_len", 1 << 30, rlh.RLH_EUNSUP)]


def structs(args):
    return rlh.KvPages(**args["kv"]), rlh.Seqs(**args["seqs"]), rlh.AppendArgs(**args["app"]), rlh.AttnArgs(**args["att"])


@pytest.mark.parametrize("part,field,value,code", APPEND)
def test_append_refuses(part, field, value, code):
    args = good()
    args[part][field] = value
    kv, seqs, app, _ = structs(args)
    assert rlh.load().rlh_paged_append(kv, seqs, app, None, None) == code
    assert rlh.load().rlh_last_error()


@pytest.mark.parametrize("part,field,value,code", ATTN)
def test_attention_refuses(part, field, value, code):
    args = good()
    args[part][field] = value
    kv, seqs, _, att = structs(args)
    lib = rlh.load()
    assert lib.rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, None, None) == code
    assert lib.rlh_last_error()
    assert lib.rlh_paged_attn_workspace(kv, seqs, att) == 0


def test_null_and_misaligned_rest():
    lib = rlh.load()
    kv, seqs, app, att = structs(good())
    assert lib.rlh_paged_append(None, seqs, app, None, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_append(kv, None, app, None, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_append(kv, seqs, None, None, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_append(kv, seqs, app, 3, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_attn(kv, seqs, None, None, 0, None, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_attn(kv, None, att, None, 0, None, None) == rlh.RLH_EINVAL
    assert lib.rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, 2, None) == rlh.RLH_EINVAL


def test_empty_batches_do_nothing():
    lib = rlh.load()
    for field in ("n_seq", "n_rows"):
        args = good()
        args["seqs"][field] = 0
        kv, seqs, app, att = structs(args)
        assert lib.rlh_paged_append(kv, seqs, app, None, None) == rlh.RLH_OK
        assert lib.rlh_paged_attn(kv, seqs, att, None, 0, None, None) == rlh.RLH_OK
        assert lib.rlh_paged_attn_workspace(kv, seqs, att) == 0
    assert lib.rlh_sample_rows(rlh.F32, None, 0, 10, 10, None, None, None, None, 0, None) == rlh.RLH_OK


def test_sample_refuses():
    lib = rlh.load()

    def call(ty=rlh.F32, logits=A, rows=2, n=100, stride=100, options=2 * A, u=3 * A, tokens=4 * A, ws=16 * A, size=1 << 40):
        return lib.rlh_sample_rows(ty, logits, rows, n, stride, options, u, tokens, ws, size, None)

    assert call(ty=rlh.Q8_0) == rlh.RLH_EUNSUP
    for bad in (dict(n=0), dict(n=(1 << 21) + 1, stride=1 << 22), dict(logits=None), dict(logits=A + 2), dict(stride=99),
                dict(stride=(1 << 32) + 1), dict(options=None), dict(options=A + 8), dict(u=None), dict(u=A + 2),
                dict(tokens=None), dict(tokens=A + 1)):
        assert call(**bad) == rlh.RLH_EINVAL, bad
    assert call(rows=1 << 23) == rlh.RLH_EUNSUP
    assert call(rows=1 << 20, n=1 << 20, stride=1 << 20) == rlh.RLH_EUNSUP
    if rlh.sample_rows_workspace(2, 100):
        assert call(ws=None) == rlh.RLH_EINVAL
        assert call(size=rlh.sample_rows_workspace(2, 100) - 1) == rlh.RLH_EINVAL
        assert call(ws=A + 8) == rlh.RLH_EINVAL


def _has_gpu():
    try:
        import torch

        return torch.cuda.device_count() > 0
    except Exception:
        return False


@pytest.mark.skipif(_has_gpu(), reason="checks the no-GPU error path")
def test_fails_loudly_without_gpu():
    lib = rlh.load()
    kv, seqs, app, att = structs(good())
    assert lib.rlh_paged_append(kv, seqs, app, None, None) == rlh.RLH_EDEVICE
    assert b"no HIP device" in lib.rlh_last_error()
    assert lib.rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, None, None) == rlh.RLH_EDEVICE
    assert lib.rlh_sample_rows(rlh.F32, A, 2, 100, 100, 2 * A, 3 * A, 4 * A, 16 * A, 1 << 40, None) == rlh.RLH_EDEVICE


# ---- rotary frequencies ---------------------------------------------------------------

def test_rope_frequencies():
    f, m = rlh.rope_freqs(128, 1e6)
    i = np.arange(64)
    assert m == 1.0 and np.allclose(f, 1e6 ** (-2 * i / 128), rtol=1e-14, atol=0)
    g, m = rlh.rope_freqs(128, 1e6, rlh.ROPE_LINEAR, factor=3.0)
    assert m == 1.0 and np.allclose(g, f / 3, rtol=1e-14, atol=0)
    g, m = rlh.rope_freqs(128, 1e6, rlh.ROPE_BANDS, factor=4.0, orig_ctx=32768)
    turns = f * 32768 / (2 * math.pi)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1.0, rel=1e-7)
    # the blend's borders are rounded outwards to whole indices
    fast, slow = np.nonzero(turns > 32)[0], np.nonzero(turns < 1)[0]
    assert np.array_equal(g[fast], f[fast]) and np.allclose(g[slow[1:]], f[slow[1:]] / 4, rtol=1e-14, atol=0)
    assert np.all(np.diff(g / f) <= 1e-15) and np.all((g / f <= 1) & (g / f >= 0.25 - 1e-15))
    g, m = rlh.rope_freqs(64, 1e4, rlh.ROPE_BANDS, factor=1.0, orig_ctx=4096)
    assert m == 1.0 and np.allclose(g, 1e4 ** (-2 * np.arange(32) / 64), rtol=1e-14, atol=0)


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=7), dict(theta=1.0), dict(theta=math.inf), dict(theta=math.nan),
                                 dict(scaling=3), dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.nan),
                                 dict(scaling=2, factor=2.0, orig_ctx=0.0),
                                 dict(scaling=2, factor=2.0, orig_ctx=100.0, beta_fast=1.0, beta_slow=1.0),
                                 dict(scaling=2, factor=2.0, orig_ctx=100.0, beta_slow=0.0)])
def test_rope_frequencies_refuse(bad):
    args = dict(rot_dim=64, theta=1e4)
    args.update(bad)
    with pytest.raises(rlh.RlhError) as e:
        rlh.rope_freqs(**args)
    assert e.value.code == rlh.RLH_EINVAL


# ---- index rules ----------------------------------------------------------------------

@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = tmp_path_factory.mktemp("paged") / "libpaged_index_shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-o", str(out),
                    os.path.join(HERE, "paged_index_shim.cpp")], check=True)
    return ctypes.CDLL(str(out))


@pytest.mark.parametrize("a,b,kv,ok,bad", [
    (0, 1, 1, True, False), (3, 8, 5, True, False), (3, 8, 100, True, False), (5, 5, 999999, False, False),
    (3, 8, 4, False, True),          # fewer positions than rows
    (3, 8, 101, False, True),        # above max_kv
    (8, 3, 50, False, True),         # starts that fall
    (3, 14, 50, False, True),        # more than max_q rows
    (15, 21, 50, False, True),       # past n_rows
    (0xfffffff0, 2, 50, False, True), (0, 0xffffffff, 50, False, True), (3, 8, 0xffffffff, False, True)])
def test_seq_view(shim, a, b, kv, ok, bad):
    out = (ctypes.c_uint32 * 3)()
    r = shim.shim_seq_view(*[ctypes.c_uint32(v) for v in (a, b, kv, 20, 10, 100)], out)
    assert r == (1 if ok else 0) | (2 if bad else 0)
    if ok:
        assert list(out) == [a, b - a, kv] and out[0] + out[1] <= 20


def test_what_rows_see(shim):
    rng = np.random.default_rng(1)
    for _ in range(3000):
        kv = int(rng.integers(1, 40))
        pos = int(rng.integers(0, kv))
        window = int(rng.choice([0, 0, 1, 2, int(rng.integers(1, 60)), 0xffffffff, 0x80000000]))
        prefix = int(rng.choice([0, 0, 1, int(rng.integers(0, 60)), 0xffffffff]))
        sees = np.zeros(64, np.uint8)
        shim.shim_sees(pos, ctypes.c_uint32(kv), ctypes.c_uint32(window), ctypes.c_uint32(prefix),
                       sees.ctypes.data_as(ctypes.c_void_p), 64)
        j = np.arange(64)
        want = (j <= pos) & ((j > pos - window) if window else True)
        want = (want | (j < prefix)) & (j < kv)
        assert np.array_equal(sees[:kv].astype(bool), want[:kv])
        last = int(rng.integers(pos, kv))
        out = (ctypes.c_int32 * 2)()
        shim.shim_range(pos, last, ctypes.c_uint32(kv), ctypes.c_uint32(window), ctypes.c_uint32(prefix), out)
        assert 0 <= out[0] < out[1] <= kv
        for p in (pos, last):
            shim.shim_sees(p, ctypes.c_uint32(kv), ctypes.c_uint32(window), ctypes.c_uint32(prefix),
                           sees.ctypes.data_as(ctypes.c_void_p), 64)
            seen = np.nonzero(sees[:kv])[0]
            assert out[0] <= seen.min() and seen.max() < out[1]


# ---- arguments that overlap, factors out of range ---------------------------------------

@pytest.mark.parametrize("field,value", [("q_out", A), ("q_out", 2 * A + 64), ("q", A), ("k", 2 * A), ("v", A + 65536 - 16)])
def test_append_refuses_the_pool(field, value):
    args = good()
    args["app"][field] = value
    kv, seqs, app, _ = structs(args)
    assert rlh.load().rlh_paged_append(kv, seqs, app, None, None) == rlh.RLH_EINVAL
    assert b"overlap" in rlh.load().rlh_last_error()


def test_attention_refuses_overlaps():
    lib = rlh.load()
    args = good()
    args["att"]["out"] = 2 * A + 65536 - 16
    kv, seqs, _, att = structs(args)
    assert lib.rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, None, None) == rlh.RLH_EINVAL
    assert b"overlaps the pool" in lib.rlh_last_error()
    kv, seqs, _, att = structs(good())
    need = rlh.paged_attn_workspace(kv, seqs, att)
    assert need > 0
    for ws in (6 * A, 7 * A + 16, A, 2 * A + 32, 6 * A - need + 16):
        assert lib.rlh_paged_attn(kv, seqs, att, ws, 1 << 40, None, None) == rlh.RLH_EINVAL
        assert b"workspace overlaps" in lib.rlh_last_error()


@pytest.mark.parametrize("scale,cap", [(3e38, 0.0), (-3e38, 0.0), (1.0, 1e-40), (1e30, 1e-30)])
def test_attention_refuses_factors_past_f32(scale, cap):
    args = good()
    args["att"].update(scale=scale, softcap=cap)
    kv, seqs, _, att = structs(args)
    assert rlh.load().rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, None, None) == rlh.RLH_EINVAL
    assert rlh.load().rlh_paged_attn_workspace(kv, seqs, att) == 0


def test_sample_refuses_overlaps():
    lib = rlh.load()
    need = rlh.sample_rows_workspace(2, 100)
    assert need > 0

    def call(logits=A, options=2 * A, u=3 * A, tokens=4 * A, ws=16 * A):
        return lib.rlh_sample_rows(rlh.F32, logits, 2, 100, 100, options, u, tokens, ws, 1 << 40, None)

    for bad in (dict(ws=A), dict(ws=2 * A), dict(ws=3 * A), dict(ws=4 * A), dict(ws=A - need + 16), dict(tokens=A + 796),
                dict(tokens=2 * A + 4), dict(tokens=3 * A + 4)):
        assert call(**bad) == rlh.RLH_EINVAL, bad
        assert b"overlap" in lib.rlh_last_error()


@pytest.mark.parametrize("n_seq,n_rows", [(65535, 6), (2, (1 << 23)), (2, (1 << 19) + 1)])
def test_sizes_past_a_launch(n_seq, n_rows):
    """n_seq * n_head_kv and n_rows * n_head beyond what a launch holds."""
    args = good()
    args["kv"].update(n_head_kv=64, n_pages=1)
    args["att"]["n_head"] = args["app"]["n_head"] = 64
    args["seqs"].update(n_seq=n_seq, n_rows=n_rows)
    kv, seqs, app, att = structs(args)
    assert rlh.load().rlh_paged_attn(kv, seqs, att, 16 * A, 1 << 40, None, None) == rlh.RLH_EUNSUP
    assert rlh.load().rlh_paged_append(kv, seqs, app, None, None) == rlh.RLH_EUNSUP
