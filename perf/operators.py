"""Timed cases of the operators for decoding with several candidates over the
fp32 KV cache: attention of a tree of drafted tokens, the decode attention step
that sums each row's attention weights, eviction of cache rows by those sums,
beam search's selection, and the in-place reordering of per-slot state.

``own`` selects what ``run`` does: the plain torch form of the operator, or the
calls of the library's entry points (include/gncx_llm_core.h).
"""
import ctypes
import math

import torch

own = False

_lib = None


def _library():
    """The library as a program sets it up once: stream-ordered calls on torch's current stream."""
    global _lib
    if _lib is None:
        from gncx_b200 import core

        lib = core.load()
        lib.gncx_set_synchronous(0)
        # torch's default stream is CUDA's legacy stream, whose explicit handle is 1
        lib.gncx_set_stream(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream or 1))
        core.check(lib)
        _lib = lib
    return _lib


def _done(lib, status):
    if status != 0:
        from gncx_b200 import core

        core.check(lib)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # speculative decoding, a short chat on a small model: launch latency counts
        {"name": "tree_small", "op": "tree", "nh": 16, "nkv": 8, "hd": 128, "pos0": 511, "n_tok": 5, "window": 0},
        # an ordinary verification step of an 8B-shaped layer, odd sizes
        {"name": "tree_4k", "op": "tree", "nh": 32, "nkv": 8, "hd": 128, "pos0": 4097, "n_tok": 33, "window": 0},
        # sliding-window layer, narrow heads, a long sequence of which the window alone counts
        {"name": "tree_window", "op": "tree", "nh": 16, "nkv": 4, "hd": 64, "pos0": 20001, "n_tok": 25, "window": 1024},
        # the widest tree over the longest cache: bandwidth and arithmetic together
        {"name": "tree_32k", "op": "tree", "nh": 32, "nkv": 8, "hd": 128, "pos0": 32768, "n_tok": 64, "window": 0},
        # one decode step with weight sums, cache at a small budget
        {"name": "step_small", "op": "step", "nh": 16, "nkv": 8, "hd": 128, "pos": 511},
        # the step over a long cache that is about to be cut down
        {"name": "step_32k", "op": "step", "nh": 32, "nkv": 8, "hd": 128, "pos": 32767},
        # steady state: one row over the budget after each token
        {"name": "evict_one", "op": "evict", "nkv": 8, "hd": 128, "n_rows": 4097, "n_keep": 4096, "n_recent": 256},
        # after a long prompt: a quarter of the rows stays
        {"name": "evict_32k", "op": "evict", "nkv": 8, "hd": 128, "n_rows": 32768, "n_keep": 8192, "n_recent": 1024},
        # beam search over the 151936-token vocabulary, the usual width
        {"name": "beam_4", "op": "beam", "n_beam": 4, "vocab": 151936, "n_out": 8, "finished": 0},
        # the widest beam, twice as many candidates as beams, some hypotheses ended
        {"name": "beam_64", "op": "beam", "n_beam": 64, "vocab": 151936, "n_out": 128, "finished": 9},
        # the accepted path of a 33-token tree, K and V of 28 layers, 4 KB a row
        {"name": "accept_33", "op": "reorder", "n_states": 56, "n_slots": 33, "row": 1024, "rows": 1, "path": True},
        # the caches of 8 beams, 1024 generated positions, K and V of 8 layers
        {"name": "reorder_8", "op": "reorder", "n_states": 16, "n_slots": 8, "row": 1024, "rows": 1024, "path": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "step", "evict", "beam", "reorder"])
    if op in ("tree", "step"):
        hd = rng.choice([64, 80, 128, 128, 256])
        nkv = rng.choice([1, 2, 4] if hd == 256 else [1, 2, 4, 8])
        nh = nkv * rng.choice([1, 2, 3, 4])
        if op == "step":
            return {"op": op, "nh": nh, "nkv": nkv, "hd": hd, "pos": _log_int(rng, 1, 32767)}
        pos0 = _log_int(rng, 1, 32768)
        window = rng.choice([0, 0, _log_int(rng, 16, 8192)])
        return {"op": op, "nh": nh, "nkv": nkv, "hd": hd, "pos0": pos0, "n_tok": _log_int(rng, 1, 64), "window": window}
    if op == "evict":
        n_rows = _log_int(rng, 64, 32768)
        n_keep = rng.choice([n_rows - 1, _log_int(rng, 16, n_rows - 1)])
        return {"op": op, "nkv": rng.choice([1, 2, 4, 8]), "hd": rng.choice([64, 80, 128]), "n_rows": n_rows,
                "n_keep": n_keep, "n_recent": rng.randint(0, n_keep // 2)}
    if op == "beam":
        n_beam = _log_int(rng, 1, 64)
        return {"op": op, "n_beam": n_beam, "vocab": _log_int(rng, 1000, 151936), "n_out": rng.choice([n_beam, 2 * n_beam]),
                "finished": rng.randint(0, n_beam // 2)}
    path = rng.random() < 0.5
    row = rng.choice([256, 500, 512, 1024])
    if path:
        return {"op": op, "n_states": rng.randint(1, 56), "n_slots": _log_int(rng, 2, 64), "row": row, "rows": 1, "path": True}
    return {"op": op, "n_states": rng.randint(1, 16), "n_slots": _log_int(rng, 2, 8), "row": row, "rows": _log_int(rng, 1, 1024), "path": False}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)  # small integer inputs

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale

    s = dict(case)
    op = case["op"]
    if op == "tree":
        n, rows = case["n_tok"], case["pos0"] + case["n_tok"]
        s["q"] = normal(n, case["nh"], case["hd"], scale=1.5)
        s["k"] = normal(rows, case["nkv"], case["hd"])
        s["v"] = normal(rows, case["nkv"], case["hd"])
        # node 0 continues the sequence; every later node hangs below an earlier one
        up = (torch.rand(n, generator=h) * torch.arange(n)).floor().int()
        up[0] = -1
        s["parents"] = up.cuda()
        s["out"] = torch.empty(n, case["nh"], case["hd"], device="cuda")
    elif op == "step":
        rows = case["pos"] + 1
        s["q"] = normal(case["nh"], case["hd"], scale=1.5)
        s["k_new"], s["v_new"] = normal(case["nkv"], case["hd"]), normal(case["nkv"], case["hd"])
        s["k"] = normal(rows, case["nkv"], case["hd"])
        s["v"] = normal(rows, case["nkv"], case["hd"])
        s["weight"] = torch.rand(case["nkv"], rows, device="cuda", generator=g)
        s["positions"] = torch.arange(rows, dtype=torch.int32, device="cuda").repeat(case["nkv"], 1)
        s["out"] = torch.empty(case["nh"], case["hd"], device="cuda")
    elif op == "evict":
        rows = case["n_rows"]
        s["k"] = normal(rows, case["nkv"], case["hd"])
        s["v"] = normal(rows, case["nkv"], case["hd"])
        # sums of attention weights: many small ones, a few heavy
        s["weight"] = torch.rand(case["nkv"], rows, device="cuda", generator=g).pow(8) * 40
        s["positions"] = torch.arange(rows, dtype=torch.int32, device="cuda").repeat(case["nkv"], 1)
        s["weight_out"] = torch.empty(case["nkv"], case["n_keep"], device="cuda")
        s["positions_out"] = torch.empty(case["nkv"], case["n_keep"], dtype=torch.int32, device="cuda")
    elif op == "beam":
        b = case["n_beam"]
        s["logits"] = normal(b, case["vocab"], scale=3.0)
        s["scores"] = -torch.rand(b, device="cuda", generator=g) * 3
        ended = torch.zeros(b, dtype=torch.int32)
        ended[torch.randperm(b, generator=h)[: case["finished"]]] = 1
        s["finished"] = ended.cuda()
        s["eos"] = 2
        s["out_scores"] = torch.empty(case["n_out"], device="cuda")
        s["out_ints"] = torch.empty(3, case["n_out"], dtype=torch.int32, device="cuda")
    else:
        n = case["n_slots"]
        s["state"] = normal(case["n_states"], n, case["rows"], case["row"])
        index = torch.randint(0, n, (n,), generator=h)
        if case["path"]:  # an ascending path of about a quarter of the nodes; the rest stays
            depth = max(1, n // 4)
            index = torch.full((n,), -1)
            index[:depth] = torch.randperm(n, generator=h)[:depth].sort().values
        s["index"] = index.int().cuda()
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"tree": _plain_tree, "step": _plain_step, "evict": _plain_evict, "beam": _plain_beam,
            "reorder": _plain_reorder}[s["op"]](s)


def _run_own(s):
    lib = _library()

    def p(name):
        return s[name].data_ptr()

    op = s["op"]
    if op == "tree":
        _done(lib, lib.gncx_attention_tree(p("q"), p("k"), p("v"), p("parents"), s["pos0"], s["n_tok"], s["nh"], s["nkv"],
                                           s["hd"], s["hd"] ** -0.5, s["window"], p("out"), None, 0))
        return s["out"]
    if op == "step":
        _done(lib, lib.gncx_mqa_attention_step_weights(
            p("q"), p("k_new"), p("v_new"), p("k"), p("v"), s["pos"], s["pos"], s["nh"], s["nkv"], s["hd"],
            s["hd"] ** -0.5, 1, p("out"), p("weight"), p("positions"), s["pos"] + 1, None, 0))
        return {"out": s["out"], "weight": s["weight"], "positions": s["positions"], "k": s["k"], "v": s["v"]}
    if op == "evict":
        _done(lib, lib.gncx_kv_evict(p("k"), p("v"), p("weight"), p("positions"), s["n_rows"], s["n_rows"], s["n_keep"],
                                     s["n_rows"] - s["n_recent"], s["nkv"], s["hd"], p("weight_out"),
                                     p("positions_out"), s["n_keep"], None, 0))
        return {"weight": s["weight_out"], "positions": s["positions_out"], "k": s["k"], "v": s["v"]}
    if op == "beam":
        ints = p("out_ints")
        _done(lib, lib.gncx_beam_select(p("logits"), p("scores"), p("finished"), s["n_beam"], s["vocab"], s["eos"],
                                        s["n_out"], p("out_scores"), ints, ints + 4 * s["n_out"], ints + 8 * s["n_out"],
                                        None, 0))
        return {"scores": s["out_scores"], "parents_tokens_finished": s["out_ints"]}
    slot = s["rows"] * s["row"] * 4
    _done(lib, lib.gncx_state_reorder(p("state"), s["n_states"], s["n_slots"] * slot, s["n_slots"], slot, slot, p("index")))
    return s["state"]


def _plain_tree(s):
    n, nh, nkv, hd, pos0 = s["n_tok"], s["nh"], s["nkv"], s["hd"], s["pos0"]
    # which drafted rows lie on each node's path: powers of (1 + parent relation)
    up = (s["parents"].long()[:, None] == torch.arange(n, device="cuda")).double()
    path = torch.linalg.matrix_power(up + torch.eye(n, device="cuda", dtype=torch.float64), n) > 0
    depth = path.sum(1) - 1
    seen = torch.cat([torch.ones(n, pos0, dtype=torch.bool, device="cuda"), path], 1)
    if s["window"] > 0:
        at = torch.cat([torch.arange(pos0, device="cuda"), pos0 + depth])
        seen &= (pos0 + depth)[:, None] - at < s["window"]
    q = s["q"].view(n, nkv, nh // nkv, hd).permute(1, 2, 0, 3)
    k = s["k"].permute(1, 2, 0)[:, None]
    v = s["v"].permute(1, 0, 2)[:, None]
    x = (q @ k) * hd ** -0.5
    x = x.masked_fill(~seen, float("-inf"))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)) @ v
    s["out"].copy_(o.permute(2, 0, 1, 3).reshape(n, nh, hd))
    return s["out"]


def _plain_step(s):
    nh, nkv, hd, pos = s["nh"], s["nkv"], s["hd"], s["pos"]
    s["k"][pos], s["v"][pos] = s["k_new"], s["v_new"]
    s["positions"][:, pos] = pos
    s["weight"][:, pos] = 0
    q = s["q"].view(nkv, nh // nkv, hd)
    x = (q @ s["k"].permute(1, 2, 0)) * hd ** -0.5
    e = torch.exp(x - x.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    s["out"].copy_((w @ s["v"].permute(1, 0, 2)).reshape(nh, hd))
    s["weight"] += w.sum(1)
    return {"out": s["out"], "weight": s["weight"], "positions": s["positions"], "k": s["k"], "v": s["v"]}


def _plain_evict(s):
    nkv, rows, keep = s["nkv"], s["n_rows"], s["n_keep"]
    w, pos = s["weight"], s["positions"]
    # protected rows first, then by weight, equal ones by row: two stable sorts
    by_weight = w.sort(dim=1, descending=True, stable=True).indices
    late = (pos >= rows - s["n_recent"]).gather(1, by_weight)
    order = by_weight.gather(1, late.int().sort(dim=1, descending=True, stable=True).indices)
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(1, order[:, :keep], True)
    # hole i of the first n_keep rows takes the i-th kept row behind them
    most = min(keep, rows - keep)
    hole = (~kept[:, :keep]).int().sort(dim=1, descending=True, stable=True).indices[:, :most]
    mover = kept[:, keep:].int().sort(dim=1, descending=True, stable=True).indices[:, :most] + keep
    moves = torch.arange(most, device="cuda") < kept[:, keep:].sum(1, keepdim=True)
    mover = torch.where(moves, mover, hole)
    head = torch.arange(nkv, device="cuda")[:, None].expand_as(hole)
    s["weight_out"].copy_(w[:, :keep])
    s["weight_out"].scatter_(1, hole, w.gather(1, mover))
    s["positions_out"].copy_(pos[:, :keep])
    s["positions_out"].scatter_(1, hole, pos.gather(1, mover))
    s["k"][hole, head] = s["k"][mover, head]
    s["v"][hole, head] = s["v"][mover, head]
    return {"weight": s["weight_out"], "positions": s["positions_out"], "k": s["k"], "v": s["v"]}


def _plain_beam(s):
    b, n, eos = s["n_beam"], s["n_out"], s["eos"]
    ended = s["finished"] != 0
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    best, token = s["logits"].sort(dim=1, descending=True, stable=True)  # equal logits: lowest token first
    m = min(n, s["vocab"])
    best, token = best[:, :m].double(), token[:, :m]
    score = s["scores"].double()[:, None] + (best - total)
    # an ended hypothesis goes on as itself, with its end token and its score
    first = torch.arange(m, device="cuda") == 0
    score = torch.where(ended[:, None], torch.where(first, s["scores"].double()[:, None], -math.inf), score)
    token = torch.where(ended[:, None], torch.full_like(token, eos), token)
    score, at = score.view(-1).sort(descending=True, stable=True)  # equal scores: lowest beam first
    score, at = score[:n], at[:n]
    none = score == -math.inf
    parent = at // m
    token = token.reshape(-1)[at]
    s["out_scores"].copy_(score)
    s["out_ints"][0] = parent.masked_fill(none, -1)
    s["out_ints"][1] = token.masked_fill(none, -1)
    s["out_ints"][2] = ((ended[parent] | (token == eos)) & ~none).int()
    return {"scores": s["out_scores"], "parents_tokens_finished": s["out_ints"]}


def _plain_reorder(s):
    i = s["index"].long()
    i = torch.where(i < 0, torch.arange(s["n_slots"], device="cuda"), i)
    s["state"].copy_(s["state"][:, i])
    return s["state"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "tree":
        prefix = min(case["pos0"], case["window"]) if case["window"] else case["pos0"]
        n, qo = case["n_tok"], case["n_tok"] * case["nh"] * case["hd"]
        return {"bytes": (prefix + n) * case["nkv"] * case["hd"] * 8 + 8 * qo + 4 * n, "flops": 4 * qo * (prefix + 1)}
    if op == "step":
        t, kv = case["pos"] + 1, case["nkv"] * case["hd"]
        return {"bytes": 8 * t * kv + 8 * kv + 8 * case["nh"] * case["hd"] + 8 * case["nkv"] * t,
                "flops": 4 * t * case["nh"] * case["hd"]}
    if op == "evict":
        n, keep, late = case["n_rows"], case["n_keep"], case["n_recent"]
        # rows kept from behind the first n_keep: the newest, and their share of the others
        behind = n - keep
        moved = min(late, behind) + max(0, behind - late) * max(0, keep - late) / max(1, n - late)
        return {"bytes": case["nkv"] * (8 * n + 8 * keep + 16 * case["hd"] * moved), "flops": case["nkv"] * n}
    if op == "beam":
        live = case["n_beam"] - case["finished"]
        return {"bytes": 4 * live * case["vocab"] + 8 * case["n_beam"] + 16 * case["n_out"], "flops": 4 * live * case["vocab"]}
    n, size = case["n_slots"], case["rows"] * case["row"] * 4
    if case["path"]:  # read and write about a quarter of the slots
        return {"bytes": case["n_states"] * size * 2 * max(1, n // 4) + 4 * n, "flops": 0}
    # index[i] = i for one slot in n; the others' sources, each once
    sources = n * (1 - (1 - 1 / n) ** n)
    return {"bytes": case["n_states"] * size * (n - 1 + sources * (n - 1) / n) + 4 * n, "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tree":
        up, n, pos0 = s["parents"].tolist(), case["n_tok"], case["pos0"]
        group, w = case["nh"] // case["nkv"], case["window"]
        out = torch.empty(n, case["nh"], case["hd"], dtype=torch.float64, device="cuda")
        k, v, q = s["k"].double(), s["v"].double(), s["q"].double()
        for i in range(n):
            chain = [i]
            while up[chain[0]] >= 0:
                chain.insert(0, up[chain[0]])
            first = max(0, pos0 + len(chain) - w) if w else 0  # lowest position seen
            rows = torch.tensor([pos0 + c for j, c in enumerate(chain) if pos0 + j >= first], device="cuda")
            ki = torch.cat([k[first:pos0], k[rows]]).repeat_interleave(group, 1)
            vi = torch.cat([v[first:pos0], v[rows]]).repeat_interleave(group, 1)
            x = (ki * q[i]).sum(-1) / math.sqrt(case["hd"])
            out[i] = (torch.softmax(x, 0)[..., None] * vi).sum(0)
        return out
    if op == "step":
        k, v = s["k"].double(), s["v"].double()
        k[-1], v[-1] = s["k_new"].double(), s["v_new"].double()
        weight = s["weight"].double()
        weight[:, -1] = 0
        out = torch.empty(case["nh"], case["hd"], dtype=torch.float64, device="cuda")
        for a in range(case["nh"]):
            c = a // (case["nh"] // case["nkv"])
            p = torch.softmax((k[:, c] * s["q"][a].double()).sum(-1) / math.sqrt(case["hd"]), 0)
            out[a] = (p[:, None] * v[:, c]).sum(0)
            weight[c] += p
        return {"out": out, "weight": weight, "positions": None, "k": None, "v": None}
    if op == "beam":
        lp = torch.log_softmax(s["logits"].double(), 1) + s["scores"].double()[:, None]
        ended = s["finished"].bool()
        lp[ended] = -math.inf
        lp[ended, 0] = s["scores"].double()[ended]
        return {"scores": lp.view(-1).sort(descending=True).values[: case["n_out"]], "parents_tokens_finished": None}
    return None
