"""The work by which the quantised operators are measured: rows of activations in 8 bits and the
products over 8-bit and 4-bit weights, as a program calls them that runs a decoder's projections and
feed-forwards from quantised weights.

  norm8    sum = x + delta; y = sum * rsqrt(mean(sum^2) + eps) * gain; the sum, and y in 8 bits (or
           without a delta y alone)
  glu8     h = g' * sigmoid(alpha g') * (u' + offset) of rows [g : u], in 8 bits
  linear8  out = (rows . values^T) * row scale * feature scale (+ add)
  linear4  out = (a . (codes - 8) group scale) * feature scale (+ add)

A row in 8 bits is e4m3 numbers q with one float32 number s, q s being what it stands for: s is the
row's largest magnitude (1e-30 at least) over 448.  A 4-bit weight is a code 0..15; eight codes of
neighbouring k lie in an int32, those of even k in its low half, those of odd k in its high half, the
lowest k in the lowest bits of each; every `group` of them shares an e4m3 scale, every output feature
has a float32 scale besides.  Sizes are those of `crucible_b200/config/presets.py` (the 120M shape and
the ones of width 2,048 and 4,096); `draw` takes others of the same ranges, odd ones among them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
TOP = 448.0
LEAST = 1e-30
EPS = 1e-5
ALPHA, OFFSET = 1.702, 1.0


def listed():
    return [
        # one decoded token of the 120M shape: the norm ahead of a projection
        {"name": "norm8 token", "op": "norm8", "rows": 1, "width": 768, "delta": "f32"},
        # a 2,048-token prompt of width 4,096, the sublayer's result still to be added
        {"name": "norm8 prompt", "op": "norm8", "rows": 2048, "width": 4096, "delta": "bf16"},
        # a capped gated pair between two products, 8 decoded tokens, sums in 32 bits
        {"name": "glu8 batch", "op": "glu8", "rows": 8, "width": 2048, "dtype": "f32", "limit": 7.0},
        # the feed-forward of a 2,048-token prompt at 14,336 features
        {"name": "glu8 prompt", "op": "glu8", "rows": 2048, "width": 14336, "dtype": "bf16", "limit": 0.0},
        # one decoded token: queries, keys and values of 32 and 8 heads of 128
        {"name": "linear8 token", "op": "linear8", "rows": 1, "n": 6144, "k": 4096, "out": "bf16", "add": False},
        # 64 decoded tokens: the feed-forward's second product, added into the residual
        {"name": "linear8 batch", "op": "linear8", "rows": 64, "n": 4096, "k": 14336, "out": "f32", "add": True},
        # a prompt portion of odd sizes all through
        {"name": "linear8 ragged", "op": "linear8", "rows": 701, "n": 5631, "k": 1000, "out": "bf16", "add": False},
        # a 2,048-token prompt: one half of the feed-forward's first product
        {"name": "linear8 prompt", "op": "linear8", "rows": 2048, "n": 14336, "k": 4096, "out": "bf16", "add": False},
        # one decoded token: both halves of the feed-forward's first product
        {"name": "linear4 token", "op": "linear4", "rows": 1, "n": 28672, "k": 4096, "group": 64,
         "dtype": "bf16", "out": "bf16", "add": False},
        # 8 decoded tokens: the logits over 128,256 tokens
        {"name": "linear4 logits", "op": "linear4", "rows": 8, "n": 128256, "k": 4096, "group": 128,
         "dtype": "bf16", "out": "f32", "add": False},
        # 33 rows in 32 bits, added into the residual, small groups
        {"name": "linear4 batch f32", "op": "linear4", "rows": 33, "n": 2048, "k": 8192, "group": 32,
         "dtype": "f32", "out": "f32", "add": True},
        # a 2,048-token prompt: the feed-forward's second product, added into the residual
        {"name": "linear4 prompt", "op": "linear4", "rows": 2048, "n": 4096, "k": 14336, "group": 64,
         "dtype": "bf16", "out": "f32", "add": True},
    ]


MOST_PRODUCT = 2048 * 14336 * 4096       # multiply-adds of the largest listed product


def _size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm8", "glu8", "linear8", "linear4"))
    if op == "norm8":
        return {"op": op, "rows": _size(rng, 1, 4096), "width": _size(rng, 64, 8192),
                "delta": rng.choice(("none", "f32", "bf16"))}
    if op == "glu8":
        return {"op": op, "rows": _size(rng, 1, 2048), "width": _size(rng, 64, 14336),
                "dtype": rng.choice(("f32", "bf16")), "limit": rng.choice((0.0, 7.0))}
    n, k = _size(rng, 64, 32768), _size(rng, 64, 16384)
    rows = min(_size(rng, 1, 4096), max(1, MOST_PRODUCT // (n * k)))
    out = rng.choice(("f32", "bf16"))
    case = {"op": op, "rows": rows, "n": n, "k": k, "out": out, "add": out == "f32" and rng.random() < 0.5}
    if op == "linear4":
        case["group"] = rng.choice((32, 64, 128))
        case["k"] = max(case["group"], k // case["group"] * case["group"])
        case["dtype"] = rng.choice(("f32", "bf16", "bf16"))
    return case


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _uniform(gen, low, high, *shape):
    return torch.rand(*shape, generator=gen, device=DEV, dtype=torch.float32) * (high - low) + low


def _padded(values):
    """The same values in rows that begin 16 bytes (or a multiple) apart."""
    rows, width = values.shape
    wide = torch.zeros(rows, -(-width // 16) * 16, dtype=values.dtype, device=values.device)
    wide[:, :width] = values
    return wide[:, :width]


def _as_rows8(y):
    """Rows in 8 bits: (e4m3 [T, K], float32 [T])."""
    scale = y.abs().amax(dim=1).clamp_min(LEAST) / TOP
    return (y / scale[:, None]).clamp(-TOP, TOP).to(E4M3), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op, rows = case["op"], case["rows"]
    state = dict(case)
    if op == "norm8":
        width = case["width"]
        # a residual whose features differ in size, some of them by much
        size = torch.exp(0.5 * _normal(gen, width))
        state["x"] = _normal(gen, rows, width) * size
        state["gain"] = 1.0 + 0.1 * _normal(gen, width)
        if case["delta"] != "none":
            state["delta_rows"] = (0.3 * _normal(gen, rows, width) * size).to(FLOATS[case["delta"]])
            state["sum"] = torch.empty_like(state["x"])
    elif op == "glu8":
        state["both"] = (2.0 * _normal(gen, rows, 2 * case["width"])).to(FLOATS[case["dtype"]])
    if op in ("norm8", "glu8"):
        state["q"] = _padded(torch.zeros(rows, case["width"], device=DEV).to(E4M3).view(torch.uint8)).view(E4M3)
        state["s"] = torch.empty(rows, device=DEV)
        return state
    n, k = case["n"], case["k"]
    if case["add"]:
        state["add_rows"] = _normal(gen, rows, n)
    state["y"] = torch.empty(rows, n, dtype=FLOATS[case["out"]], device=DEV)
    if op == "linear8":
        # values as they come out of a rounding to 8 bits: each row's largest is 448
        values, state["s"] = _as_rows8(_normal(gen, rows, k))
        state["q"] = _padded(values.view(torch.uint8)).view(E4M3)
        values, state["feature_scale"] = _as_rows8(_normal(gen, n, k) * 0.02)
        state["values"] = _padded(values.view(torch.uint8)).view(E4M3)
        return state
    state["a"] = _normal(gen, rows, k).to(FLOATS[case["dtype"]])
    words = torch.empty(n, k // 8, dtype=torch.int32, device=DEV)
    for at in range(0, n, 16384):                 # (codes of a bell's shape, some at either end)
        m = min(16384, n - at)
        codes = (torch.round(_normal(gen, m, k // 8, 8) * 2.8).clamp(-8, 7) + 8).to(torch.int32)
        word = torch.zeros(m, k // 8, dtype=torch.int32, device=DEV)
        for i in range(8):
            word |= codes[:, :, i] << (4 * (i // 2) + 16 * (i % 2))
        words[at:at + m] = word
    state["codes"] = words
    state["group_scale"] = _uniform(gen, 100.0, 448.0, n, k // case["group"]).to(E4M3)
    state["feature_scale"] = _uniform(gen, 2e-5, 4e-5, n)
    return state


def _plain_glu(state):
    g, u = state["both"].float().chunk(2, dim=1)
    if state["limit"] > 0:
        g, u = g.clamp(max=state["limit"]), u.clamp(-state["limit"], state["limit"])
        return g / (1.0 + torch.exp(-ALPHA * g)) * (u + OFFSET)
    return g / (1.0 + torch.exp(-g)) * u


def _plain_weights4(state):
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=DEV)
    codes = (state["codes"][:, :, None] >> shifts) & 15
    n = codes.shape[0]
    scale = state["group_scale"].float()[:, :, None]
    return ((codes - 8).float().view(n, -1, state["group"]) * scale).view(n, -1)


def _plain_out(state, products):
    y = products * state["feature_scale"]
    if state["op"] == "linear8":
        y = y * state["s"][:, None]
    if state["add"]:
        y = y + state["add_rows"]
    return y.to(FLOATS[state["out"]])


def run(state):
    op = state["op"]
    if own:
        from crucible_b200.ops import quantized
        if op == "norm8":
            if state["delta"] == "none":
                quantized.add_rmsnorm8(state["x"], None, state["gain"], EPS, state["q"], state["s"])
                return [state["q"], state["s"]]
            quantized.add_rmsnorm8(state["x"], state["delta_rows"], state["gain"], EPS, state["q"], state["s"],
                                   sum_out=state["sum"])
            return [state["sum"], state["q"], state["s"]]
        if op == "glu8":
            if state["limit"] > 0:
                quantized.glu8(state["both"], state["q"], state["s"], state["limit"], ALPHA, OFFSET)
            else:
                quantized.glu8(state["both"], state["q"], state["s"])
            return [state["q"], state["s"]]
        add = state["add_rows"] if state["add"] else None
        if op == "linear8":
            w = quantized.Weights8(state["values"], state["feature_scale"])
            quantized.linear8(state["q"], state["s"], w, state["y"], add=add)
        else:
            w = quantized.Weights4(state["codes"], state["group_scale"], state["feature_scale"])
            quantized.linear4(state["a"], w, state["y"], add=add)
        return state["y"]
    if op == "norm8":
        x = state["x"] if state["delta"] == "none" else state["x"] + state["delta_rows"].float()
        y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * state["gain"]
        return [*_as_rows8(y)] if state["delta"] == "none" else [x, *_as_rows8(y)]
    if op == "glu8":
        return [*_as_rows8(_plain_glu(state))]
    if op == "linear8":
        return _plain_out(state, state["q"].float() @ state["values"].float().t())
    return _plain_out(state, state["a"].float() @ _plain_weights4(state).t())


def _work8(rows, width):
    return rows * width + 4 * rows


def work(case):
    op, rows = case["op"], case["rows"]
    size = {"none": 0, "f32": 4, "bf16": 2}
    if op == "norm8":
        values = rows * case["width"]
        moved = values * (4 if case["delta"] == "none" else 8 + size[case["delta"]])
        return {"bytes": moved + 4 * case["width"] + _work8(rows, case["width"]), "flops": 7 * values}
    if op == "glu8":
        values = rows * case["width"]
        return {"bytes": 2 * values * size[case["dtype"]] + _work8(rows, case["width"]), "flops": 8 * values}
    n, k = case["n"], case["k"]
    moved = rows * n * (size[case["out"]] + (4 if case["add"] else 0)) + 4 * n
    if op == "linear8":
        moved += _work8(rows, k) + n * k
    else:
        moved += rows * k * size[case["dtype"]] + n * k // 2 + n * (k // case["group"])
    return {"bytes": moved, "flops": 2 * rows * n * k}


def _exact_rows8(y):
    """Each row over its scale, every number to the nearest of e4m3 (ties to the even one): three bits
    behind the leading one, the smallest step 2^-9."""
    scale = torch.maximum(y.abs().max(dim=1).values, torch.tensor(LEAST, dtype=torch.float64, device=DEV)) / TOP
    v = y / scale.unsqueeze(1)
    power = torch.frexp(v).exponent.clamp_min(-5) - 4
    q = torch.ldexp(torch.round(torch.ldexp(v, -power)), power)
    return [q.clamp(-TOP, TOP).to(torch.float32).to(E4M3), scale.to(torch.float32)]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm8":
        x = state["x"].double()
        if case["delta"] != "none":
            x = x.add(state["delta_rows"].double())
        length = torch.sqrt(x.pow(2).sum(dim=1) / case["width"] + EPS)
        rows8 = _exact_rows8(x / length.unsqueeze(1) * state["gain"].double())
        return [*rows8] if case["delta"] == "none" else [x, *rows8]
    if op == "glu8":
        g, u = (t.double() for t in state["both"].split(case["width"], dim=1))
        if case["limit"] > 0:
            g = torch.minimum(g, torch.full_like(g, case["limit"]))
            u = torch.maximum(torch.minimum(u, torch.full_like(u, case["limit"])), torch.full_like(u, -case["limit"]))
            return _exact_rows8(g * torch.sigmoid(ALPHA * g) * (u + OFFSET))
        return _exact_rows8(g * torch.sigmoid(g) * u)
    rows = state["q"].double() * state["s"].double().unsqueeze(1) if op == "linear8" else state["a"].double()
    out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEV)
    for at in range(0, case["n"], 4096):
        to = min(case["n"], at + 4096)
        if op == "linear8":
            w = state["values"][at:to].double()
        else:
            words = state["codes"][at:to]
            w = torch.empty(to - at, case["k"], dtype=torch.float64, device=DEV)
            for i in range(8):
                w[:, i::8] = (torch.bitwise_and(words >> (4 * (i // 2) + 16 * (i % 2)), 15) - 8).double()
            w.mul_(state["group_scale"][at:to].double().repeat_interleave(case["group"], dim=1))
        w.mul_(state["feature_scale"][at:to].double().unsqueeze(1))
        torch.mm(rows, w.t(), out=out[:, at:to])
    if case["add"]:
        out.add_(state["add_rows"].double())
    return out
