"""The operators of a batched serving step and the cases whose speed is
measured: rows of many sequences appended to a paged key/value cache (norms
and position rotation on the way), attention over that cache (prompts, single
tokens, mixed batches, a prefix shared by the whole batch) and one token
sampled per row.

`run` with `own` false computes them in elementary torch operations in 32 bits
(64 for far angles and for sampling, where values lie next to a border), with
`own` true it calls the binding `rlh` as a server's loop does. Heads are those
of the Qwen3 shapes the package knows (16, 32 or 64 query heads over 8 KV
heads of 128), the vocabulary is theirs, prompts and contexts run up to their
window.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}  # ggml ids


# ---- cases ------------------------------------------------------------------

def listed():
    """op append: `seqs` sequences that each bring up to `q` new rows.
    op attn: `seqs` sequences with up to `q` new rows, up to `ctx` positions in
    all; `shared` of them common to the batch. op sample: `rows` rows of
    logits. `spread`: how unequal the sequences are."""
    return [
        # a server's decode step, half-precision projections, interleaved
        # pairs over half of the head, positions far out (scaled frequencies)
        {"name": "append 93 tokens far", "op": "append", "heads": 32, "kv": 8, "dim": 128, "page": 32, "type": "f16",
         "in": "f16", "seqs": 93, "q": 1, "ctx": 130001, "spread": 1.0, "layout": "inter", "rot": 64, "norm": False,
         "far": True},
        # several prompts at once on the largest model, rows from f32 products
        {"name": "append prompts 9503", "op": "append", "heads": 64, "kv": 8, "dim": 128, "page": 64, "type": "bf16",
         "in": "f32", "seqs": 4, "q": 2900, "ctx": 4000, "spread": 0.6, "layout": "half", "rot": 128, "norm": True,
         "far": False},
        # one conversation's next token: nothing but latency
        _attn("decode 1 at 777", 16, 8, "bf16", 16, seqs=1, q=1, ctx=777),
        # a server's decode step over conversations of unequal length
        _attn("decode 61 ragged", 32, 8, "bf16", 16, seqs=61, q=1, ctx=8191, spread=1.0),
        # few long documents on the largest model: split over the length
        _attn("decode 3 at 40000", 64, 8, "f16", 64, seqs=3, q=1, ctx=40000, spread=0.1),
        # one long prompt on the largest model
        _attn("prompt 4096", 64, 8, "bf16", 64, seqs=1, q=4096, ctx=4096),
        # chunks of prompts beside single tokens, capped scores and a window
        _attn("mixed capped window", 32, 8, "f16", 32, seqs=12, q=700, ctx=5003, spread=1.0, mixed=True, cap=30.0,
              window=1024),
        # ragged prompts whose first part sees itself whole, distance bias
        _attn("prompts prefix bias", 16, 8, "bf16", 16, seqs=5, q=2111, ctx=2111, spread=0.7, prefix=True, bias=True),
        # a batch under one long system prompt
        _attn("shared 4096 by 64", 32, 8, "bf16", 16, seqs=64, q=1, ctx=4096 + 511, spread=1.0, shared=4096),
        # the same on the largest model with a small batch of drafts
        _attn("shared 16384 by 24", 64, 8, "f16", 64, seqs=24, q=3, ctx=16384 + 300, spread=1.0, shared=16384),
        # one row with the command line's defaults, and a server's batch with
        # options of every kind
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "in": "f32", "mix": "default"},
        {"name": "sample 192", "op": "sample", "rows": 192, "vocab": 151936, "in": "f32", "mix": "every"},
    ]


def _attn(name, heads, kv, kind, page, seqs, q, ctx, spread=0.0, mixed=False, cap=0.0, window=0, prefix=False,
          bias=False, shared=0, dim=128):
    return {"name": name, "op": "attn", "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind, "seqs": seqs,
            "q": q, "ctx": ctx, "spread": spread, "mixed": mixed, "cap": cap, "window": window, "prefix": prefix,
            "bias": bias, "shared": shared}


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Every operator over batch sizes 1 to 128, new rows 1 to 4096, contexts
    1 to 40000, the head groupings of the package's shapes and their
    neighbours, both cache types, all masks and options."""
    op = rng.choice(["append", "attn", "attn", "attn", "shared", "sample"])
    if op == "sample":
        rows = _log_uniform(rng, 1, 192)
        return {"op": "sample", "rows": rows, "vocab": _log_uniform(rng, 1000, 151936),
                "in": rng.choice(["f32", "bf16", "f16"]), "mix": rng.choice(["default", "every"])}
    heads, kv = rng.choice([(16, 8), (32, 8), (64, 8), (40, 8), (28, 4), (8, 8), (12, 1)])
    dim = rng.choice([128, 128, 64])
    case = {"heads": heads, "kv": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
            "type": rng.choice(["bf16", "f16"]), "spread": rng.choice([0.0, 0.5, 1.0])}
    if op == "append":
        total = _log_uniform(rng, 1, 7000)
        seqs = min(total, _log_uniform(rng, 1, 128))
        far = rng.random() < 0.3
        q = max(1, total // seqs)
        return {"op": "append", **case, "in": rng.choice(["f32", "bf16", "f16"]), "seqs": seqs, "q": q,
                "ctx": _log_uniform(rng, max(q, 100), 131072 if far else 8192), "layout": rng.choice(["half", "inter"]),
                "rot": rng.choice([dim, dim // 2]), "norm": rng.random() < 0.6, "far": far}
    if op == "shared":
        shared = case["page"] * _log_uniform(rng, 2, 8192 // case["page"])
        seqs = _log_uniform(rng, 2, 64)
        return {"op": "attn", **case, "seqs": seqs, "q": rng.choice([1, 1, 2, 5]),
                "ctx": shared + _log_uniform(rng, 8, 1000), "mixed": False, "cap": 0.0, "window": 0, "prefix": False,
                "bias": False, "shared": shared}
    kind = rng.choice(["decode", "prompt", "mixed"])
    cap, window = rng.choice([0.0, 0.0, 30.0]), rng.choice([0, 0, 0, 333, 1024])
    if kind == "decode":
        ctx = _log_uniform(rng, 1, 40000)
        seqs = _log_uniform(rng, 1, max(1, min(128, 200000 // ctx)))
        q = 1
    else:
        q = _log_uniform(rng, 2, 4096)
        ctx = min(q + (0 if rng.random() < 0.5 else _log_uniform(rng, 1, 4096)), 5000)
        seqs = _log_uniform(rng, 1, max(1, min(16, 8000 // ctx)))
    case = {"op": "attn", **case, "seqs": seqs, "q": q, "ctx": ctx, "mixed": kind == "mixed", "cap": cap,
            "window": window, "prefix": kind == "prompt" and rng.random() < 0.3, "bias": rng.random() < 0.25,
            "shared": 0}
    while work(case)["flops"] > 2.7e11:
        case["ctx"] -= case["q"] // 2
        case["q"] -= case["q"] // 2
    return case


def _lengths(case):
    """(new rows, positions in all) of each sequence: whole numbers that
    follow from the case alone."""
    n, rng = case["seqs"], random.Random(case["seqs"] * 7919 + case["ctx"] * 31 + case["q"])
    new, length = [], []
    for i in range(n):
        short = 1.0 if i == 0 else math.exp(-2.0 * case["spread"] * rng.random())
        q = max(1, int(case["q"] * (1.0 if case["q"] <= 8 else short)))
        if case.get("mixed") and i % 3:
            q = 1
        base = case.get("shared", 0)
        own_part = max(q, int((case["ctx"] - base) * short))
        new.append(q)
        length.append(base + own_part)
    return new, length


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * case["vocab"] * (4 if case["in"] == "f32" else 2),
                "flops": 4 * case["rows"] * case["vocab"]}
    new, length = _lengths(case)
    h, g, d = case["heads"], case["kv"], case["dim"]
    rows = sum(new)
    if case["op"] == "append":
        size = 4 if case["in"] == "f32" else 2
        return {"bytes": rows * (h + 2 * g) * d * (size + 2), "flops": rows * (h + g) * d * 6}
    shared = case["shared"]
    read = shared
    pairs = 0
    for q, n in zip(new, length):
        first = n - q
        low = 0
        if case["window"] and not case["prefix"]:
            low = max(0, first - case["window"] + 1)
        read += n - max(low, shared)
        for i in range(q):
            p = first + i
            seen = p + 1 if not case["window"] else min(p + 1, case["window"])
            if case["prefix"]:
                pre = _prefix_len(q, n)
                seen = max(seen, min(n, pre)) if not case["window"] else seen + max(0, min(pre, p + 1 - seen)) \
                    + max(0, pre - (p + 1))
            pairs += seen
    return {"bytes": 2 * rows * h * d * 2 + 2 * read * g * d * 2, "flops": 4 * pairs * h * d}


def _prefix_len(q, n):
    return max(0, n - q) + (q * 3) // 8


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, seed, g)
    new, length = _lengths(case)
    h, kv, d, page, kind = case["heads"], case["kv"], case["dim"], case["page"], TYPES[case["type"]]
    n, rows = len(new), sum(new)
    shared = case.get("shared", 0)
    keep = page * (-(-max(length) // page))
    if case["op"] == "append":
        # only the pages that hold new rows take part: the others of the
        # table stand for pages of the pool that this step leaves alone
        first = [(t - q) // page for q, t in zip(new, length)]
    else:
        first = [shared // page] * n
    counts = [-(-t // page) - f for t, f in zip(length, first)]
    n_pages = sum(counts) + shared // page + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    stride = keep // page
    table = torch.zeros((n, stride), dtype=torch.int32, device="cuda")
    at = shared // page
    for i in range(n):
        table[i, first[i]:first[i] + counts[i]] = order[at:at + counts[i]]
        at += counts[i]
    shape = (n_pages, kv, page, d)
    state = {"case": case, "rows": rows, "max_q": max(new), "max_kv": max(length), "n_pages": n_pages,
             "q_start": torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda"),
             "kv_len": torch.tensor(length, dtype=torch.int32, device="cuda"), "table": table,
             "k": torch.randn(shape, generator=g, device="cuda").to(kind),
             "v": torch.randn(shape, generator=g, device="cuda").to(kind)}
    if case["op"] == "append":
        width = (h + 2 * kv) * d
        # the three products' rows side by side, as one product writes them
        state["qkv"] = (1.7 * torch.randn((rows, width), generator=g, device="cuda")).to(TYPES[case["in"]])
        state["q_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
        state["k_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if case["norm"] else None
        state["freqs"], state["magnitude"] = _frequencies(case["rot"], 1e6, 4.0 if case["far"] else 1.0, 32768)
        state["q_out"] = torch.zeros((rows, h, d), dtype=kind, device="cuda")
        return state
    state["q"] = (1.3 * torch.randn((rows, h, d), generator=g, device="cuda")).to(kind)
    state["out"] = torch.zeros((rows, h, d), dtype=kind, device="cuda")
    state["shared_table"] = order[:shared // page].contiguous() if shared else None
    if shared:
        table[:, :shared // page] = state["shared_table"]
    state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], dtype=torch.float32,
                                   device="cuda") if case["bias"] else None
    state["prefix"] = torch.tensor([_prefix_len(q, t) for q, t in zip(new, length)], dtype=torch.int32,
                                   device="cuda") if case["prefix"] else None
    return state


def _frequencies(rot, theta, factor, trained):
    """f_i = theta^(-2i/rot); with a factor, the slow ones (less than one turn
    over the trained window) are divided by it, the fast ones (32 turns) kept,
    the rest blended, and the rotated values grow by 0.1 ln(factor) + 1."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    f = theta ** (-2.0 * i / rot)
    if factor == 1.0:
        return f, 1.0

    def at(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _prepare_sample(case, seed, g):
    rows, n = case["rows"], case["vocab"]
    logits = 2.2 * torch.randn((rows, n), generator=g, device="cuda")
    # a few tokens that the model finds likely
    likely = torch.randint(0, n, (rows, 24), generator=g, device="cuda")
    logits.scatter_(1, likely, 7 + 5 * torch.rand((rows, 24), generator=g, device="cuda"))
    rng = random.Random(seed)
    sets = [(0.7, 40, 0.95, 0.0)]
    if case["mix"] == "every":
        sets += [(1.0, 0, 0.9, 0.0), (0.8, 100, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (1.2, 0, 1.0, 0.0),
                 (0.9, 1000, 0.8, 0.02), (0.6, 20, 0.95, 0.0)]
    pick = [sets[i % len(sets)] for i in range(rows)]
    rng.shuffle(pick)
    options = torch.tensor(pick, dtype=torch.float32, device="cuda")
    options[:, 1] = torch.tensor([p[1] for p in pick], dtype=torch.int32, device="cuda").view(torch.float32)
    return {"case": case, "logits": logits.to(TYPES[case["in"]]), "options": options.contiguous(),
            "u": torch.rand(rows, generator=g, device="cuda"),
            "token": torch.zeros(rows, dtype=torch.int32, device="cuda")}


# ---- one pass ---------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attn": _own_attn, "sample": _own_sample}[op](state)
    return {"append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}[op](state)


def _binding():
    if "rlh" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "llama.rs_amd"))
    import rlh

    return rlh


def _own_batch(rlh, state):
    case = state["case"]
    kv = rlh.KvPages(TYPE_IDS[case["type"]], case["kv"], case["dim"], case["page"], state["n_pages"],
                     state["k"].data_ptr(), state["v"].data_ptr())
    seqs = rlh.Seqs(len(state["kv_len"]), state["rows"], state["max_q"], state["max_kv"], state["table"].shape[1],
                    state["q_start"].data_ptr(), state["kv_len"].data_ptr(), state["table"].data_ptr())
    return kv, seqs


def _own_append(state):
    rlh = _binding()
    case = state["case"]
    kv, seqs = _own_batch(rlh, state)
    h, g, d = case["heads"], case["kv"], case["dim"]
    qkv, q_out = state["qkv"], state["q_out"]
    at, size = qkv.data_ptr(), qkv.element_size()
    norm = case["norm"]
    args = rlh.AppendArgs(TYPE_IDS[case["in"]], h, at, at + h * d * size, at + (h + g) * d * size, qkv.stride(0),
                          qkv.stride(0), qkv.stride(0), state["q_norm"].data_ptr() if norm else None,
                          state["k_norm"].data_ptr() if norm else None, 1e-6, state["magnitude"],
                          state["freqs"].data_ptr(), case["rot"], 1 if case["layout"] == "inter" else 0,
                          q_out.data_ptr(), q_out.stride(0))
    rlh.paged_append(kv, seqs, args, None, torch.cuda.current_stream().cuda_stream)
    return [q_out, state["k"], state["v"]]


def _own_attn(state):
    rlh = _binding()
    case = state["case"]
    kv, seqs = _own_batch(rlh, state)
    q, out = state["q"], state["out"]
    shared, slopes, prefix = state["shared_table"], state["slopes"], state["prefix"]
    args = rlh.AttnArgs(case["heads"], case["window"], q.data_ptr(), out.data_ptr(), q.stride(0), out.stride(0),
                        case["dim"] ** -0.5, case["cap"], slopes.data_ptr() if case["bias"] else None,
                        prefix.data_ptr() if case["prefix"] else None,
                        shared.data_ptr() if case["shared"] else None, case["shared"])
    if "workspace" not in state:  # a server makes it once, for its largest batch
        state["workspace"] = torch.empty(max(16, rlh.paged_attn_workspace(kv, seqs, args)), dtype=torch.uint8,
                                         device="cuda")
    ws = state["workspace"]
    rlh.paged_attn(kv, seqs, args, ws.data_ptr(), ws.numel(), None, torch.cuda.current_stream().cuda_stream)
    return out


def _own_sample(state):
    rlh = _binding()
    logits, token = state["logits"], state["token"]
    rows, n = logits.shape
    if "workspace" not in state:
        state["workspace"] = torch.empty(max(16, rlh.sample_rows_workspace(rows, n)), dtype=torch.uint8, device="cuda")
    ws = state["workspace"]
    rlh.sample_rows(TYPE_IDS[state["case"]["in"]], logits.data_ptr(), rows, n, logits.stride(0),
                    state["options"].data_ptr(), state["u"].data_ptr(), token.data_ptr(), ws.data_ptr(), ws.numel(),
                    torch.cuda.current_stream().cuda_stream)
    return token


# ---- the plain forms --------------------------------------------------------

def _row_places(state):
    """Of each new row: its sequence and its position."""
    start, length = state["q_start"].long(), state["kv_len"].long()
    seq = torch.repeat_interleave(torch.arange(len(length), device="cuda"), start[1:] - start[:-1],
                                  output_size=state["rows"])
    row = torch.arange(state["rows"], device="cuda")
    return seq, length[seq] - (start[1:] - start[:-1])[seq] + row - start[seq]


def _plain_append(state):
    case = state["case"]
    h, g, d, page, rot = case["heads"], case["kv"], case["dim"], case["page"], case["rot"]
    rows = state["rows"]
    seq, pos = _row_places(state)
    x = state["qkv"].float().view(rows, h + 2 * g, d)
    q, k, v = x[:, :h], x[:, h:h + g], x[:, h + g:]
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * state["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * state["k_norm"]
    angle = pos.double()[:, None] * state["freqs"][None, :]
    cos = (torch.cos(angle) * state["magnitude"]).float()[:, None, :]
    sin = (torch.sin(angle) * state["magnitude"]).float()[:, None, :]

    def rotate(t):
        t = t.clone()
        if case["layout"] == "half":
            a, b = t[..., :rot // 2].clone(), t[..., rot // 2:rot].clone()
            t[..., :rot // 2] = a * cos - b * sin
            t[..., rot // 2:rot] = b * cos + a * sin
        else:
            a, b = t[..., 0:rot:2].clone(), t[..., 1:rot:2].clone()
            t[..., 0:rot:2] = a * cos - b * sin
            t[..., 1:rot:2] = b * cos + a * sin
        return t

    kind = TYPES[case["type"]]
    state["q_out"].copy_(rotate(q).to(kind))
    where = state["table"][seq, pos // page].long()
    state["k"][where, :, pos % page] = rotate(k).to(kind)
    state["v"][where, :, pos % page] = v.to(kind)
    return [state["q_out"], state["k"], state["v"]]


def _visible(case, i, j, length, prefix):
    """Whether the row at position i sees position j of its sequence."""
    see = j <= i
    if case["window"]:
        see = see & (j > i - case["window"])
    if prefix is not None:
        see = see | (j < prefix)
    return see & (j < length)


def _plain_attn(state):
    case = state["case"]
    h, g, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    n, most_q, most = len(state["kv_len"]), state["max_q"], state["max_kv"]
    group = h // g
    start, length = state["q_start"].long(), state["kv_len"].long()
    new = start[1:] - start[:-1]
    j = torch.arange(most, device="cuda")
    where = state["table"][:, :].long()[:, j // page]
    # [sequence, KV head, position, dim]
    k = state["k"][where, :, (j % page)[None, :]].permute(0, 2, 1, 3).float().contiguous()
    v = state["v"][where, :, (j % page)[None, :]].permute(0, 2, 1, 3).float()
    v = torch.where((j[None, :] < length[:, None])[:, None, :, None], v, 0.0).contiguous()
    seq, pos = _row_places(state)
    local = torch.arange(state["rows"], device="cuda") - start[seq]
    q = torch.zeros((n, most_q, h, d), device="cuda")
    q[seq, local] = state["q"].float()
    q = q.view(n, most_q, g, group, d).permute(0, 2, 3, 1, 4).reshape(n, g, group * most_q, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, g, group, most_q, most) * d ** -0.5
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    i = (length - new)[:, None] + torch.arange(most_q, device="cuda")[None, :]
    away = (j[None, None, :] - i[:, :, None])
    if case["bias"]:
        s = s + state["slopes"].view(1, g, group, 1, 1) * away[:, None, None].float()
    prefix = state["prefix"].long()[:, None, None] if case["prefix"] else None
    see = _visible(case, i[:, :, None], j[None, None, :], length[:, None, None], prefix)
    s = torch.where(see[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, g, group * most_q, most), v).view(n, g, group, most_q, d)
    o = o / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most_q, h, d)
    state["out"].copy_(o[seq, local].to(TYPES[case["type"]]))
    return state["out"]


def _plain_sample(state):
    x = state["logits"].double()
    rows, n = x.shape
    options = state["options"]
    heat, top_p, min_p = (options[:, c].double()[:, None] for c in (0, 2, 3))
    top_k = options[:, 1].contiguous().view(torch.int32).long()[:, None]
    top_k = torch.where((top_k == 0) | (top_k > n), n, top_k)
    first = torch.argmax(x, dim=1)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(heat > 0, heat, 1.0))
    before = torch.cumsum(w, 1) - w
    keep = torch.arange(n, device="cuda")[None, :] < top_k
    keep &= (before < top_p * w.sum(1, keepdim=True)) | (top_p <= 0) | (top_p >= 1)
    keep &= w >= min_p
    mass = torch.zeros_like(x).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    running = torch.cumsum(mass, 1)
    drawn = (running <= state["u"].double()[:, None] * running[:, -1:]).sum(1)
    state["token"].copy_(torch.where(heat[:, 0] > 0, drawn, first))
    return state["token"]


# ---- from the definitions, in 64 bits ---------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, state)


def _exact_append(case, state):
    """One sequence after the other, pairs as complex numbers."""
    h, g, d, page, rot = case["heads"], case["kv"], case["dim"], case["page"], case["rot"]
    new, length = _lengths(case)
    q_out, pool_k, pool_v = state["q_out"].double(), state["k"].double(), state["v"].double()
    at = 0
    for s, (rows, total) in enumerate(zip(new, length)):
        pos = torch.arange(total - rows, total, device="cuda")
        x = state["qkv"][at:at + rows].double()
        turn = torch.polar(torch.full((), float(state["magnitude"]), dtype=torch.float64, device="cuda"),
                           torch.outer(pos.double(), state["freqs"]))
        parts = []
        for lo, heads, weight in ((0, h, state["q_norm"]), (h * d, g, state["k_norm"])):
            t = x[:, lo:lo + heads * d].reshape(rows, heads, d).clone()
            if weight is not None:
                t = t / torch.sqrt((t ** 2).sum(-1, keepdim=True) / d + 1e-6) * weight.double()
            if case["layout"] == "half":
                z = torch.complex(t[..., :rot // 2].contiguous(), t[..., rot // 2:rot].contiguous()) * turn[:, None]
                t[..., :rot // 2], t[..., rot // 2:rot] = z.real, z.imag
            else:
                z = torch.complex(t[..., 0:rot:2].contiguous(), t[..., 1:rot:2].contiguous()) * turn[:, None]
                t[..., 0:rot:2], t[..., 1:rot:2] = z.real, z.imag
            parts.append(t)
        q_out[at:at + rows] = parts[0]
        pages = state["table"][s].long()[torch.div(pos, page, rounding_mode="floor")]
        slot = pos - page * torch.div(pos, page, rounding_mode="floor")
        pool_k[pages, :, slot] = parts[1]
        pool_v[pages, :, slot] = x[:, (h + g) * d:].reshape(rows, g, d)
        at += rows
    return [q_out, pool_k, pool_v]


def _exact_attn(case, state):
    """One sequence and one KV head after the other."""
    h, g, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    new, length = _lengths(case)
    group = h // g
    out = torch.zeros((sum(new), h, d), dtype=torch.float64, device="cuda")
    at = 0
    for s, (rows, total) in enumerate(zip(new, length)):
        pages = state["table"][s, :-(-total // page)].long()
        j = torch.arange(total, device="cuda", dtype=torch.float64)
        i = torch.arange(total - rows, total, device="cuda", dtype=torch.float64)[:, None]
        ahead = j[None, :] - i
        hide = ahead > 0
        if case["window"]:
            hide |= ahead <= -case["window"]
        if case["prefix"]:
            hide &= ~(j < _prefix_len(rows, total))[None, :]
        for head in range(g):
            k = state["k"][pages, head].reshape(-1, d)[:total].double()
            v = state["v"][pages, head].reshape(-1, d)[:total].double()
            for m in range(head * group, (head + 1) * group):
                score = state["q"][at:at + rows, m].double() @ k.T / math.sqrt(d)
                if case["cap"]:
                    score = case["cap"] * torch.tanh(score / case["cap"])
                if case["bias"]:
                    score = score + state["slopes"][m].double() * ahead
                score = score.masked_fill(hide, -math.inf)
                out[at:at + rows, m] = torch.softmax(score, dim=-1).nan_to_num(0.0) @ v
        at += rows
    return out


def _exact_sample(case, state):
    """Row by row, with the sorted list cut step by step."""
    x, u = state["logits"].double(), state["u"].double()
    options = state["options"].cpu()
    whole = state["options"][:, 1].contiguous().view(torch.int32).cpu()
    tokens = []
    for r in range(case["rows"]):
        heat, top_k, top_p, min_p = float(options[r, 0]), int(whole[r]), float(options[r, 2]), float(options[r, 3])
        value, index = torch.sort(x[r], descending=True, stable=True)
        if heat <= 0:
            tokens.append(index[0])
            continue
        p = torch.softmax(value / heat, dim=0)
        count = len(p) if top_k == 0 else min(top_k, len(p))
        if 0 < top_p < 1:
            count = min(count, int((torch.cumsum(p, 0) < top_p).sum()) + 1)
        count = min(count, int((p >= min_p * p[0]).sum()))
        chosen, by_index = torch.sort(index[:count])
        running = torch.cumsum(p[:count][by_index], 0)
        tokens.append(chosen[torch.searchsorted(running, u[r] * running[-1], right=True).clamp(max=count - 1)])
    return torch.stack(tokens).to(torch.int32)
