"""The operators that edit a paged key/value cache, and the cases whose speed is
measured: masks and positions of trees of drafted tokens, attention of such
trees over the cache, keeping an accepted branch (the walk and the move of its
rows), the attention weight that each cached position gathers, and eviction of
those that gathered least (the choice and the move of what stays).

`run` with `own` false computes them in elementary torch operations, in 32
bits, with `own` true it calls the binding `rlh` as a server's loop does. Heads
are those of the Qwen3 shapes the package knows (16, 32 or 64 query heads over 8
KV heads of 128), the vocabulary is theirs, contexts run up to their window.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TYPE_IDS = {"f16": 1, "bf16": 30}  # ggml ids
VOCAB = 151936
DECAY = 0.97


# ---- cases ------------------------------------------------------------------

def listed():
    """op masks, tree, commit: `seqs` sequences with a tree of up to `nodes`
    drafted tokens each. op tree, mass, evict: up to `ctx` positions in all;
    `shared` of them common to the batch. op mass: the weights of the last
    `nodes` rows. op evict: `budget` positions stay, the first `first` and the
    last `last` among them. `spread`: how unequal the sequences are."""
    return [
        # one conversation's draft: nothing but latency
        {"name": "masks 1 x 26", "op": "masks", "seqs": 1, "nodes": 26, "spread": 0.0},
        # a server's drafts of one step
        {"name": "masks 120 x 63", "op": "masks", "seqs": 120, "nodes": 63, "spread": 0.6},
        # one conversation, a few drafted tokens on the smallest model
        _tree("tree 1 x 7 at 777", 16, "bf16", 16, seqs=1, nodes=7, ctx=777),
        # a server's conversations of unequal length
        _tree("tree 16 x 26 ragged", 32, "bf16", 16, seqs=16, nodes=26, ctx=8191, spread=1.0),
        # few long documents, wide trees on the largest model
        _tree("tree 4 x 63 at 30000", 64, "f16", 64, seqs=4, nodes=63, ctx=30011, spread=0.1),
        # small trees under one long system prompt, capped scores and a window
        _tree("tree 24 x 9 shared", 32, "bf16", 32, seqs=24, nodes=9, ctx=4096 + 700, spread=1.0, shared=4096,
              cap=30.0, window=4500),
        # the end of a step: the accepted branches are walked and kept
        _commit("commit 1 x 26", 16, "bf16", 16, seqs=1, nodes=26, ctx=777),
        _commit("commit 96 x 63", 32, "f16", 32, seqs=96, nodes=63, ctx=8191),
        # what a server's single tokens attend to, added to the running weights
        _mass("mass 61 ragged", 32, "bf16", 16, seqs=61, nodes=1, ctx=8191, spread=1.0),
        # what the last rows of long prompts attend to: decides what is kept
        _mass("mass 3 x 32 at 20000", 64, "f16", 64, seqs=3, nodes=32, ctx=20011, spread=0.3),
        # one long document is cut down, and a server's batch by a quarter
        _evict("evict 1 of 40000", 8, "bf16", 16, seqs=1, ctx=40000, budget=4096, first=4, last=256),
        _evict("evict 24 ragged", 8, "f16", 64, seqs=24, ctx=8191, budget=2048, first=16, last=512, spread=0.5),
    ]


def _tree(name, heads, kind, page, seqs, nodes, ctx, kv=8, dim=128, spread=0.0, shared=0, cap=0.0, window=0):
    return {"name": name, "op": "tree", "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind, "seqs": seqs,
            "nodes": nodes, "ctx": ctx, "spread": spread, "shared": shared, "cap": cap, "window": window}


def _commit(name, heads, kind, page, seqs, nodes, ctx, kv=8, dim=128, spread=0.6):
    return {"name": name, "op": "commit", "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind,
            "seqs": seqs, "nodes": nodes, "ctx": ctx, "spread": spread}


def _mass(name, heads, kind, page, seqs, nodes, ctx, kv=8, dim=128, spread=0.0, cap=0.0, window=0):
    return {"name": name, "op": "mass", "heads": heads, "kv": kv, "dim": dim, "page": page, "type": kind, "seqs": seqs,
            "nodes": nodes, "ctx": ctx, "spread": spread, "cap": cap, "window": window}


def _evict(name, kv, kind, page, seqs, ctx, budget, first, last, dim=128, spread=0.0):
    return {"name": name, "op": "evict", "kv": kv, "dim": dim, "page": page, "type": kind, "seqs": seqs, "ctx": ctx,
            "budget": budget, "first": first, "last": last, "spread": spread}


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Every operator over batches of 1 to 128 sequences, trees of 1 to 150
    nodes, contexts from the tree alone to 40000, the head groupings of the
    package's shapes and their neighbours, both types, caps and windows."""
    op = rng.choice(["masks", "tree", "tree", "tree", "commit", "mass", "mass", "evict", "evict"])
    spread = rng.choice([0.0, 0.5, 1.0])
    nodes = _log_uniform(rng, 1, 150)
    if op == "masks":
        return {"op": op, "seqs": _log_uniform(rng, 1, 128), "nodes": nodes, "spread": spread}
    heads, kv = rng.choice([(16, 8), (32, 8), (64, 8), (40, 8), (28, 4), (8, 8), (12, 1)])
    case = {"op": op, "kv": kv, "dim": rng.choice([128, 128, 64]), "page": rng.choice([16, 32, 64, 128]),
            "type": rng.choice(["bf16", "f16"]), "spread": spread}
    if op == "evict":
        ctx = _log_uniform(rng, 50, 40000)
        budget = max(1, int(ctx * rng.choice([0.1, 0.25, 0.5, 0.9, 1.2])))
        first, last = rng.randrange(budget // 4 + 1), rng.randrange(budget // 4 + 1)
        return {**case, "seqs": _log_uniform(rng, 1, max(1, min(64, 60000 // ctx))), "ctx": ctx, "budget": budget,
                "first": first, "last": last}
    case["heads"], case["nodes"] = heads, nodes
    if op == "commit":
        return {**case, "seqs": _log_uniform(rng, 1, 96), "ctx": _log_uniform(rng, nodes, 8192)}
    case["cap"], case["window"] = rng.choice([0.0, 0.0, 30.0]), rng.choice([0, 0, 333, 1024])
    if op == "mass":
        ctx = _log_uniform(rng, nodes, 40000)
        rows = 200000 // ctx * 32 // nodes
        return {**case, "ctx": ctx, "seqs": _log_uniform(rng, 1, max(1, min(128, 200000 // ctx, rows)))}
    shared = case["page"] * _log_uniform(rng, 2, 4096 // case["page"]) if rng.random() < 0.3 else 0
    ctx = shared + _log_uniform(rng, nodes, 20000)
    seqs = _log_uniform(rng, 1, max(1, min(64, 6000000 // (ctx * nodes), 110000 // ctx)))
    return {**case, "ctx": ctx, "seqs": seqs, "shared": shared}


def _lengths(case):
    """(new rows, positions in all) of each sequence: whole numbers that
    follow from the case alone."""
    rng = random.Random(case["seqs"] * 7919 + case.get("ctx", 0) * 31 + case.get("nodes", 0))
    new, length = [], []
    for i in range(case["seqs"]):
        short = 1.0 if i == 0 else math.exp(-2.0 * case["spread"] * rng.random())
        q = max(1, int(case.get("nodes", 1) * (1.0 if case["op"] == "mass" else math.sqrt(short))))
        base = case.get("shared", 0)
        new.append(q)
        length.append(base + max(q, int((case.get("ctx", q) - base) * short)))
    return new, length


def _words(new):
    return (max(new) + 63) // 64


def work(case):
    new, length = _lengths(case)
    rows = sum(new)
    if case["op"] == "masks":
        return {"bytes": rows * (4 + 8 * _words(new) + 4), "flops": 2 * rows}
    g, d = case["kv"], case["dim"]
    if case["op"] == "commit":
        # three rows of a branch stay; parents, tokens and draws are read
        return {"bytes": 12 * rows + 3 * case["seqs"] * 2 * 2 * g * d * 2, "flops": 2 * rows}
    if case["op"] == "evict":
        moved = sum(max(0, case["budget"] - case["first"]) for n in length if n > case["budget"])
        return {"bytes": 4 * g * sum(n for n in length if n > case["budget"]) + moved * g * (2 * 2 * d * 2 + 12),
                "flops": 2 * g * sum(length)}
    h, shared, window = case["heads"], case.get("shared", 0), case["window"]
    pairs, read = 0, shared
    for q, n in zip(new, length):
        first = n - q
        low = max(0, first + 1 - window) if window else 0
        read += n - max(low, shared)
        pairs += q * (first - low + 1)
    if case["op"] == "mass":
        return {"bytes": rows * h * (d * 2 + 4) + read * g * (d * 2 + 8), "flops": 2 * pairs * h * d}
    return {"bytes": 2 * rows * h * d * 2 + 2 * read * g * d * 2, "flops": 4 * pairs * h * d}


# ---- inputs -----------------------------------------------------------------

def _trees(new, seed):
    """Of each row its parent within its sequence; the first has none."""
    rng = random.Random(seed * 2654435761 + len(new))
    parents = []
    for q in new:
        parents += [-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, q)]
    return parents


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new, length = _lengths(case)
    rows, n = sum(new), len(new)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    state = {"case": case, "rows": rows, "max_q": max(new), "max_kv": max(length), "words": _words(new),
             "q_start": ints([sum(new[:i]) for i in range(n + 1)]), "kv_len": ints(length)}
    if case["op"] in ("masks", "tree", "commit"):
        state["parents"] = ints(_trees(new, seed))
    if case["op"] == "masks":
        state["base"] = torch.randint(0, 40000, (n,), generator=g, device="cuda", dtype=torch.int32)
        state["masks"] = torch.zeros((rows, state["words"]), dtype=torch.int64, device="cuda")
        state["positions"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        return state
    kv, d, page, kind = case["kv"], case["dim"], case["page"], TYPES[case["type"]]
    shared = case.get("shared", 0)
    # pages that the call takes part in: of a commit, those of the new rows
    first = [(t - q) // page if case["op"] == "commit" else shared // page for q, t in zip(new, length)]
    counts = [-(-t // page) - f for t, f in zip(length, first)]
    state["n_pages"] = sum(counts) + shared // page + 3
    order = torch.randperm(state["n_pages"], generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((n, -(-max(length) // page)), dtype=torch.int32, device="cuda")
    at = shared // page
    for i in range(n):
        table[i, first[i]:first[i] + counts[i]] = order[at:at + counts[i]]
        at += counts[i]
    state["shared_table"] = order[:shared // page].contiguous() if shared else None
    if shared:
        table[:, :shared // page] = state["shared_table"]
    state["table"] = table
    shape = (state["n_pages"], kv, page, d)
    state["k"] = torch.randn(shape, generator=g, device="cuda").to(kind)
    state["v"] = torch.randn(shape, generator=g, device="cuda").to(kind)
    return {"tree": _prepare_tree, "commit": _prepare_commit, "mass": _prepare_mass,
            "evict": _prepare_evict}[case["op"]](state, seed, g)


def _prepare_tree(state, seed, g):
    case = state["case"]
    shape = (state["rows"], case["heads"], case["dim"])
    kind = TYPES[case["type"]]
    state["q"] = (1.3 * torch.randn(shape, generator=g, device="cuda")).to(kind)
    state["out"] = torch.zeros(shape, dtype=kind, device="cuda")
    # made once per step, for the attention of every layer
    state["masks"] = _plain_masks(state)[0]
    return state


def _prepare_commit(state, seed, g):
    """Drafted tokens, and the tokens that the model drew at each node: along
    one branch they are mostly a child's."""
    rng = random.Random(seed)
    start, parents = state["q_start"].tolist(), state["parents"].tolist()
    tokens, sampled = [], []
    for a, b in zip(start, start[1:]):
        drafted = [rng.randrange(VOCAB) for _ in range(a, b)]
        for i in range(2, b - a):
            if rng.random() < 0.1:  # siblings may carry the same token
                drafted[i] = drafted[i - 1]
        drawn = [rng.randrange(VOCAB) for _ in range(a, b)]
        at = 0
        while rng.random() < 0.75:
            children = [i for i in range(at + 1, b - a) if parents[a + i] == at]
            if not children:
                break
            child = rng.choice(children)
            drawn[at] = drafted[child]
            at = min(i for i in children if drafted[i] == drafted[child])
        tokens += drafted
        sampled += drawn
    n = len(start) - 1
    for name, values in (("tokens", tokens), ("sampled", sampled)):
        state[name] = torch.tensor(values, dtype=torch.int32, device="cuda")
    # the sequences' lengths without their drafts
    state["base"] = state["kv_len"] - (state["q_start"][1:] - state["q_start"][:-1])
    state["path"] = torch.zeros((n, state["max_q"]), dtype=torch.int32, device="cuda")
    for name in ("count", "next", "new_len"):
        state[name] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return state


def _prepare_mass(state, seed, g):
    case = state["case"]
    state["q"] = (1.3 * torch.randn((state["rows"], case["heads"], case["dim"]), generator=g, device="cuda")).to(
        TYPES[case["type"]])
    state["mass"] = torch.rand((state["n_pages"], case["kv"], case["page"]), generator=g, device="cuda")
    # as the attention of the same step left them
    s = _mass_scores(state)
    seq, local = _places(state)
    lse = torch.logsumexp(s.double(), -1).float()  # [sequence, KV head, group, row]
    state["lse"] = lse.permute(0, 3, 1, 2)[seq, local].reshape(state["rows"], case["heads"]).contiguous()
    return state


def _prepare_evict(state, seed, g):
    case = state["case"]
    shape = (state["n_pages"], case["kv"], case["page"])
    mass = torch.exp(2.0 * torch.randn(shape, generator=g, device="cuda"))
    # positions that nothing attended to, and equal weights
    kind = torch.rand(shape, generator=g, device="cuda")
    mass = torch.where(kind < 0.05, 0.0, torch.where(kind < 0.3, torch.round(mass * 16) / 16, mass))
    state["mass"], state["mass_out"] = mass, torch.zeros_like(mass)
    n = case["seqs"]
    state["keep"] = torch.zeros((n, case["kv"], min(case["budget"], state["max_kv"])), dtype=torch.int32,
                                device="cuda")
    state["count"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return state


# ---- one pass ---------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"masks": _own_masks, "tree": _own_tree, "commit": _own_commit, "mass": _own_mass,
                "evict": _own_evict}[op](state)
    return {"masks": _plain_masks_run, "tree": _plain_tree, "commit": _plain_commit, "mass": _plain_mass,
            "evict": _plain_evict}[op](state)


def _binding():
    if "rlh" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "llama.rs_amd"))
    import rlh

    return rlh


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_batch(rlh, state):
    """The descriptors of the pool and of the batch, which a server keeps for
    its buffers."""
    if "batch" not in state:
        case = state["case"]
        kv = None
        if "k" in state:
            kv = rlh.KvPages(TYPE_IDS[case["type"]], case["kv"], case["dim"], case["page"], state["n_pages"],
                             state["k"].data_ptr(), state["v"].data_ptr())
        table = state.get("table")
        seqs = rlh.Seqs(case["seqs"], state["rows"], state["max_q"], state["max_kv"],
                        table.shape[1] if table is not None else 0, state["q_start"].data_ptr(),
                        state["kv_len"].data_ptr(), table.data_ptr() if table is not None else None)
        state["batch"] = (kv, seqs)
    return state["batch"]


def _own_masks(state):
    rlh = _binding()
    _, seqs = _own_batch(rlh, state)
    rlh.tree_masks(seqs, state["parents"].data_ptr(), state["base"].data_ptr(), state["masks"].data_ptr(),
                   state["words"], state["positions"].data_ptr(), None, _stream())
    return [state["masks"], state["positions"]]


def _own_tree(state):
    rlh = _binding()
    case = state["case"]
    kv, seqs = _own_batch(rlh, state)
    if "args" not in state:
        q, out, shared = state["q"], state["out"], state["shared_table"]
        state["args"] = rlh.AttnArgs(case["heads"], case["window"], q.data_ptr(), out.data_ptr(), q.stride(0),
                                     out.stride(0), case["dim"] ** -0.5, case["cap"], None, None,
                                     shared.data_ptr() if case["shared"] else None, case["shared"])
        state["workspace"] = torch.empty(max(16, rlh.tree_attn_workspace(kv, seqs, state["args"])), dtype=torch.uint8,
                                         device="cuda")
    ws = state["workspace"]
    rlh.tree_attn(kv, seqs, state["args"], state["masks"].data_ptr(), state["words"], None, ws.data_ptr(), ws.numel(),
                  None, _stream())
    return state["out"]


def _own_commit(state):
    rlh = _binding()
    kv, seqs = _own_batch(rlh, state)
    if "args" not in state:
        path = state["path"]
        state["args"] = (
            rlh.AcceptArgs(state["parents"].data_ptr(), state["tokens"].data_ptr(), state["sampled"].data_ptr(),
                           path.data_ptr(), path.shape[1], state["count"].data_ptr(), state["next"].data_ptr(),
                           state["new_len"].data_ptr()),
            rlh.MoveArgs(path.data_ptr(), path.shape[1], 0, state["count"].data_ptr(), path.shape[1],
                         state["base"].data_ptr(), None, None))
    accept, move = state["args"]
    rlh.tree_accept(seqs, accept, None, _stream())
    rlh.paged_move(kv, seqs, move, None, _stream())
    return [state["path"], state["count"], state["next"], state["new_len"], state["k"], state["v"]]


def _own_mass(state):
    rlh = _binding()
    case = state["case"]
    kv, seqs = _own_batch(rlh, state)
    if "args" not in state:
        q = state["q"]
        state["args"] = rlh.AttnArgs(case["heads"], case["window"], q.data_ptr(), None, q.stride(0), 0,
                                     case["dim"] ** -0.5, case["cap"], None, None, None, 0)
    rlh.paged_mass(kv, seqs, state["args"], state["lse"].data_ptr(), DECAY, state["mass"].data_ptr(), None, _stream())
    return state["mass"]


def _own_evict(state):
    rlh = _binding()
    case = state["case"]
    kv, seqs = _own_batch(rlh, state)
    if "args" not in state:
        keep = state["keep"]
        state["args"] = (
            rlh.EvictArgs(state["mass"].data_ptr(), case["budget"], case["first"], case["last"], keep.shape[2],
                          keep.data_ptr(), state["count"].data_ptr()),
            rlh.MoveArgs(keep.data_ptr(), keep.shape[2], 1, state["count"].data_ptr(), keep.shape[2], None,
                         state["mass"].data_ptr(), state["mass_out"].data_ptr()))
    choice, move = state["args"]
    rlh.evict_select(kv, seqs, choice, None, _stream())
    rlh.paged_move(kv, seqs, move, None, _stream())
    return [state["keep"], state["count"], state["k"], state["v"], state["mass_out"]]


# ---- the plain forms --------------------------------------------------------

def _places(state):
    """Of each new row: its sequence and its place there."""
    start = state["q_start"].long()
    seq = torch.repeat_interleave(torch.arange(len(start) - 1, device="cuda"), start[1:] - start[:-1],
                                  output_size=state["rows"])
    return seq, torch.arange(state["rows"], device="cuda") - start[seq]


def _padded_parents(state):
    """[sequence, row] -> parent; rows of their own behind a sequence's last."""
    seq, local = _places(state)
    q = state["max_q"]
    parent = torch.full((len(state["kv_len"]), q), -1, dtype=torch.long, device="cuda")
    parent[seq, local] = state["parents"].long()
    return parent


def _plain_masks(state):
    """Reachability over the parents by squaring: after k steps, 2^k edges."""
    parent = _padded_parents(state)
    q = state["max_q"]
    i = torch.arange(q, device="cuda")
    reach = ((parent[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (q - 1).bit_length())):
        reach = torch.matmul(reach, reach).clamp(max=1.0)
    see = torch.zeros((parent.shape[0], q, 64 * state["words"]), dtype=torch.long, device="cuda")
    see[:, :, :q] = reach.long()
    bit = torch.ones(64, dtype=torch.long, device="cuda") << torch.arange(64, device="cuda")
    masks = (see.view(parent.shape[0], q, state["words"], 64) * bit).sum(-1)
    seq, local = _places(state)
    return masks[seq, local], see.sum(-1)[seq, local]


def _plain_masks_run(state):
    masks, seen = _plain_masks(state)
    seq, _ = _places(state)
    state["masks"].copy_(masks)
    state["positions"].copy_(state["base"].long()[seq] + seen - 1)
    return [state["masks"], state["positions"]]


def _seen_rows(state):
    """[sequence, row, row]: whether a new row sees another, from the bits."""
    seq, local = _places(state)
    q = state["max_q"]
    bits = (state["masks"][:, :, None] >> torch.arange(64, device="cuda")) & 1
    see = torch.zeros((len(state["kv_len"]), q, q), dtype=torch.bool, device="cuda")
    see[seq, local] = bits.view(state["rows"], -1)[:, :q].bool()
    return see


def _scores(state):
    """[sequence, KV head, group, row, position] before any mask, and the
    pages and slots of the positions."""
    case = state["case"]
    h, g, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    n, most_q, most = len(state["kv_len"]), state["max_q"], state["max_kv"]
    j = torch.arange(most, device="cuda")
    where = state["table"].long()[:, j // page], (j % page)[None, :]
    k = state["k"][where[0], :, where[1]].permute(0, 2, 3, 1).float().contiguous()
    seq, local = _places(state)
    q = torch.zeros((n, most_q, h, d), device="cuda")
    q[seq, local] = state["q"].float()
    q = q.view(n, most_q, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(n, g, h // g * most_q, d)
    s = torch.matmul(q, k).view(n, g, h // g, most_q, most) * d ** -0.5
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    return s, where


def _plain_tree(state):
    case = state["case"]
    h, g, d = case["heads"], case["kv"], case["dim"]
    n, most_q, most = len(state["kv_len"]), state["max_q"], state["max_kv"]
    start, length = state["q_start"].long(), state["kv_len"].long()
    first = (length - (start[1:] - start[:-1]))[:, None, None]
    s, where = _scores(state)
    rows = _seen_rows(state)
    j = torch.arange(most, device="cuda")
    see = (j < first).expand(n, most_q, most)
    if case["window"]:
        see = see & (j >= first + rows.sum(-1, keepdim=True) - case["window"])
    drafted = (j - first).expand(n, most_q, most)
    see = see | ((drafted >= 0) & torch.gather(rows, 2, drafted.clamp(0, most_q - 1)))
    see = see & (j < length[:, None, None])
    s = torch.where(see[:, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = state["v"][where[0], :, where[1]].permute(0, 2, 1, 3).float()
    v = torch.where((j[None, :] < length[:, None])[:, None, :, None], v, 0.0).contiguous()
    o = torch.matmul(p.view(n, g, h // g * most_q, most), v).view(n, g, h // g, most_q, d)
    o = o / torch.where(total == 0, 1.0, total)
    seq, local = _places(state)
    state["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, most_q, h, d)[seq, local].to(TYPES[case["type"]]))
    return state["out"]


def _plain_move(state, index, count, base):
    """Slot base + j of each KV head takes the row of slot base + index[j],
    j < count; index: [sequence, KV head, j]. (Where, from where.)"""
    page = state["case"]["page"]
    n, g, most = index.shape
    j = torch.arange(most, device="cuda")
    to = (base.long()[:, None, None] + j).expand(n, g, most)
    to = torch.minimum(to, state["kv_len"].long()[:, None, None] - 1)  # (behind the count: any own slot)
    source = torch.where(j < count.long()[:, None, None], base.long()[:, None, None] + index.long(), to)
    table = state["table"].long()
    seq = torch.arange(n, device="cuda")[:, None, None]
    head = torch.arange(g, device="cuda")[None, :, None]
    to, source = ((table[seq, p // page], head, p % page) for p in (to, source))
    for name in ("k", "v"):
        state[name][to] = state[name][source]
    return to, source


def _plain_commit(state):
    case = state["case"]
    parent = _padded_parents(state)
    n, q = parent.shape
    seq, local = _places(state)
    token = torch.full((n, q), -1, dtype=torch.long, device="cuda")
    drawn = torch.full((n, q), -2, dtype=torch.long, device="cuda")
    token[seq, local], drawn[seq, local] = state["tokens"].long(), state["sampled"].long()
    i = torch.arange(q, device="cuda")
    up = parent.clamp(min=0)
    ok = (parent >= 0) & (token == torch.gather(drawn, 1, up))
    # of siblings with one token the first
    twin = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :])
    twin = twin & (i[None, :] < i[:, None])
    ok = (ok & ~twin.any(-1)) | (i == 0)
    for _ in range(max(1, (q - 1).bit_length())):  # all of a row's edges: twice as many each time
        ok = ok & torch.gather(ok, 1, up)
        up = torch.gather(up, 1, up)
    count = ok.sum(1)
    place = torch.where(ok, torch.cumsum(ok, 1) - 1, q)
    path = torch.zeros((n, q + 1), dtype=torch.long, device="cuda").scatter_(1, place, i.expand(n, q))[:, :q]
    path = torch.where(i < count[:, None], path, 0)
    last = torch.gather(path, 1, count[:, None] - 1)
    state["path"].copy_(path)
    state["count"].copy_(count)
    state["next"].copy_(torch.gather(drawn, 1, last)[:, 0])
    state["new_len"].copy_(state["base"] + count)
    # (row by row the places behind the count move to themselves; never past the drafts)
    _plain_move(state, path[:, None, :].expand(n, case["kv"], q), count, state["base"])
    return [state["path"], state["count"], state["next"], state["new_len"], state["k"], state["v"]]


def _mass_scores(state):
    """Scores with minus infinity where a row does not see a position."""
    case = state["case"]
    s, _ = _scores(state)
    start, length = state["q_start"].long(), state["kv_len"].long()
    new = start[1:] - start[:-1]
    j = torch.arange(state["max_kv"], device="cuda")
    i = (length - new)[:, None, None] + torch.arange(state["max_q"], device="cuda")[:, None]
    see = (j <= i) & (i < length[:, None, None])
    if case["window"]:
        see = see & (j > i - case["window"])
    return torch.where(see[:, None, None], s, -math.inf)


def _plain_mass(state):
    case = state["case"]
    g, page, n, most_q = case["kv"], case["page"], len(state["kv_len"]), state["max_q"]
    s = _mass_scores(state)
    seq, local = _places(state)
    lse = torch.zeros((n, most_q, case["heads"]), device="cuda")
    lse[seq, local] = state["lse"]
    lse = lse.view(n, most_q, g, -1).permute(0, 2, 3, 1)
    added = torch.exp(s - lse[..., None]).sum((2, 3))  # [sequence, KV head, position]
    j = torch.arange(state["max_kv"], device="cuda")
    length = state["kv_len"].long()[:, None]
    new = (state["q_start"][1:] - state["q_start"][:-1]).long()[:, None]
    live = (j < length)[:, None, :].expand(n, g, len(j))
    pages = state["table"].long()[:, j // page][:, None, :].expand(n, g, len(j))
    at = (pages, torch.arange(g, device="cuda")[None, :, None].expand(n, g, len(j)), (j % page).expand(n, g, len(j)))
    old = torch.where((j < length - new)[:, None, :], DECAY * state["mass"][at], 0.0)
    state["mass"][tuple(x[live] for x in at)] = (old + added)[live]
    return state["mass"]


def _plain_evict(state):
    case = state["case"]
    g, page, n, most = case["kv"], case["page"], len(state["kv_len"]), state["max_kv"]
    j = torch.arange(most, device="cuda")
    length = state["kv_len"].long()[:, None, None]
    mass = state["mass"][state["table"].long()[:, j // page], :, (j % page)[None, :]].permute(0, 2, 1)
    rank = torch.where((j < case["first"]) | (j >= length - case["last"]), math.inf, mass)
    rank = torch.where(j < length, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    count = length[:, 0, 0].clamp(max=case["budget"])
    kept = state["keep"].shape[2]
    c = torch.arange(kept, device="cuda")
    live = c < count[:, None, None]
    keep = torch.sort(torch.where(live, order[..., :kept], most), dim=-1).values
    state["keep"].copy_(torch.where(live, keep, 0))
    state["count"].copy_(count)
    base = torch.zeros_like(count)
    # nothing moves in a sequence that stays whole: its list counts up
    to, source = _plain_move(state, state["keep"], count, base)
    to, source = (tuple(x.expand(n, g, kept)[live.expand(n, g, kept)] for x in at) for at in (to, source))
    state["mass_out"][to] = state["mass"][source]
    return [state["keep"], state["count"], state["k"], state["v"], state["mass_out"]]


# ---- from the definitions, in 64 bits ---------------------------------------

def exact(case, seed):
    if case["op"] == "masks":
        return None  # whole numbers
    state = prepare(case, seed)
    return {"tree": _exact_tree, "commit": _exact_commit, "mass": _exact_mass, "evict": _exact_evict}[case["op"]](
        case, state)


def _keys(case, state, name, s, head, total):
    pages = state["table"][s, :-(-total // case["page"])].long()
    return state[name][pages, head].reshape(-1, case["dim"])[:total].double()


def _logits(case, q, k):
    s = q.double() @ k.T / math.sqrt(case["dim"])
    return case["cap"] * torch.tanh(s / case["cap"]) if case["cap"] else s


def _exact_tree(case, state):
    """One sequence and one head after the other; ancestors by walking up."""
    new, length = _lengths(case)
    group = case["heads"] // case["kv"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    parents, at = state["parents"].tolist(), 0
    for s, (rows, total) in enumerate(zip(new, length)):
        first = total - rows
        hide = torch.ones((rows, total), dtype=torch.bool)
        for i in range(rows):
            line, up = [], i
            while up >= 0:
                line.append(first + up)
                up = parents[at + up]
            hide[i, line] = False
            hide[i, max(0, first + len(line) - case["window"]) if case["window"] else 0:first] = False
        hide = hide.cuda()
        for m in range(case["heads"]):
            k, v = (_keys(case, state, name, s, m // group, total) for name in ("k", "v"))
            score = _logits(case, state["q"][at:at + rows, m], k).masked_fill(hide, -math.inf)
            out[at:at + rows, m] = torch.softmax(score, dim=-1) @ v
        at += rows
    return out


def _exact_commit(case, state):
    """The walk, node by node, and its rows one after the other."""
    new, length = _lengths(case)
    page = case["page"]
    k, v = state["k"].double(), state["v"].double()
    parents, tokens, sampled = (state[name].tolist() for name in ("parents", "tokens", "sampled"))
    at = 0
    for s, (rows, total) in enumerate(zip(new, length)):
        node, kept = 0, 0
        while node is not None:
            to, source = total - rows + kept, total - rows + node
            for pool in (k, v):
                pool[state["table"][s, to // page].long(), :, to % page] = pool[
                    state["table"][s, source // page].long(), :, source % page]
            kept += 1
            node = next((i for i in range(node + 1, rows) if parents[at + i] == node
                         and tokens[at + i] == sampled[at + node]), None)
        at += rows
    return [None, None, None, None, k, v]


def _exact_mass(case, state):
    new, length = _lengths(case)
    group, page = case["heads"] // case["kv"], case["page"]
    mass = state["mass"].double()
    at = 0
    for s, (rows, total) in enumerate(zip(new, length)):
        j = torch.arange(total, device="cuda")
        i = torch.arange(total - rows, total, device="cuda")[:, None]
        hide = j > i
        if case["window"]:
            hide = hide | (j <= i - case["window"])
        pages = state["table"][s].long()[torch.div(j, page, rounding_mode="floor")]
        slots = j - page * torch.div(j, page, rounding_mode="floor")
        for head in range(case["kv"]):
            k = _keys(case, state, "k", s, head, total)
            got = torch.where(j < total - rows, DECAY * mass[pages, head, slots], 0.0)
            for m in range(head * group, (head + 1) * group):
                score = _logits(case, state["q"][at:at + rows, m], k)
                p = torch.exp(score - state["lse"][at:at + rows, m].double()[:, None])
                got = got + p.masked_fill(hide, 0.0).sum(0)
            mass[pages, head, slots] = got
        at += rows
    return mass


def _exact_evict(case, state):
    """One sequence and one head after the other, by sorted (weight, place)
    pairs; rows and weights are copied."""
    _, length = _lengths(case)
    page = case["page"]
    k, v, out = state["k"].double(), state["v"].double(), state["mass_out"].double()
    k0, v0, mass = state["k"].clone(), state["v"].clone(), state["mass"]
    for s, total in enumerate(length):
        for head in range(case["kv"]):
            j = torch.arange(total, device="cuda")
            pages, slots = state["table"][s].long()[j // page], j % page
            w = mass[pages, head, slots].double()
            kept = j
            if total > case["budget"]:
                middle = j[case["first"]:total - case["last"]]
                best = torch.argsort(-w[middle], stable=True)[:case["budget"] - case["first"] - case["last"]]
                kept = torch.cat([j[:case["first"]], middle[torch.sort(best).values], j[total - case["last"]:]])
            to, at = slice(0, len(kept)), kept
            k[pages[to], head, slots[to]] = k0[pages[at], head, slots[at]].double()
            v[pages[to], head, slots[to]] = v0[pages[at], head, slots[at]].double()
            out[pages[to], head, slots[to]] = w[at]
    return [None, None, k, v, out]
