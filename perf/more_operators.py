"""The work by which the operators over a key/value cache in 4 bits are measured: writing it, attention that
reads it, and attention over the pages of it that a cheap score picks, as a program calls them that serves a decoder.

  append  q and k of the packed rows are rotated by their positions; k and v go to the cache's pages in 4 bits
          (with bounds: what each written page holds, feature by feature, is bounded anew)
  attend  o = softmax(scale q.k) v over the keys of a row's request up to the row itself (or the last `window`)
  picked  for every row and key/value head `count` pages are picked by a bound on the logits in them; attention
          over the keys of these pages alone

A key or value is held by groups of `group` features as codes 0..15 with a bfloat16 pair (step, low) and stands
for code * step + low: low is the group's least number rounded down to bfloat16, step is (largest - low) * (1 / 15)
rounded to bfloat16 (0 if it is under 1e-30), the code is (x - low) * (1 / step) rounded to the nearest.  What is
coded is the rotated row in float32, and every operation up to the code is rounded to float32 once, so that the
codes are defined to the last bit; so are the bounds.

Pages: codes uint8 [2, pages, kv heads, page tokens, dim / 2] (keys, values), scales bfloat16 [2, pages, kv
heads, page tokens, dim / group, 2].  A row's bytes are int32 words; word (dim / 64) g + w, g < 8, holds the
codes of the features 64 w + 8 k + g, and its four bits n (the lowest first) are that of k = (0, 1, 4, 5, 2, 3, 6, 7)[n].
Bounds: int8 [pages, kv heads, 2, dim] (largest, least), float32 scales [pages, kv heads].

Sizes are those of `crucible_b200/config/presets.py` (the 120M shape, 12 heads of 64 on 4; 32 heads of 128 on 8)
and generic ones; `draw` takes others of the same ranges, odd ones among them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16}
ORDER = (0, 1, 4, 5, 2, 3, 6, 7)
THETA = 500000.0
LEAST_STEP = 1e-30


def _case(name, op, dtype, heads, kv_heads, dim, group, page, requests, new, held, **more):
    given = {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "group": group,
             "page": page, "requests": requests, "lead": 0, "new": new, "held": held, "window": 0, "bounds": False,
             "rotary": dim, "neighbours": False, "count": 0}
    given.update(more)
    return given


def listed():
    return [
        # one decoded token of the 120M shape
        _case("append token", "append", "bf16", 12, 4, 64, 64, 16, 1, 1, 700),
        # 64 decoded tokens of the 8B shape, long pages whose bounds are kept
        _case("append batch", "append", "bf16", 32, 8, 128, 64, 64, 64, 1, 8000, bounds=True),
        # a 2,048-token prompt of the 8B shape
        _case("append prompt", "append", "bf16", 32, 8, 128, 64, 16, 1, 2048, 0),
        # portions behind odd contexts, half of each head rotated by neighbours, pages of 24, in 32 bits
        _case("append ragged f32", "append", "f32", 14, 2, 128, 32, 24, 7, 250, 1001, rotary=64, neighbours=True),
        # one decoded token of the 120M shape behind a short context
        _case("attend token", "attend", "bf16", 12, 4, 64, 64, 16, 1, 1, 700),
        # 64 decoded tokens of the 8B shape behind contexts of up to 8,191
        _case("attend batch", "attend", "bf16", 32, 8, 128, 64, 16, 64, 1, 8191),
        # one decoded token behind a very long context
        _case("attend long", "attend", "bf16", 32, 8, 128, 128, 64, 1, 1, 131071),
        # small portions and single tokens in 32 bits, a window, pages of 24
        _case("attend ragged f32", "attend", "f32", 14, 2, 128, 32, 24, 9, 33, 3001, lead=4, window=1000),
        # a 2,048-token prompt of the 8B shape
        _case("attend prompt", "attend", "bf16", 32, 8, 128, 64, 16, 1, 2048, 0),
        # 16 decoded tokens behind contexts of up to 32,767, 64 pages of 64 each
        _case("picked batch", "picked", "bf16", 32, 8, 128, 64, 64, 16, 1, 32767, bounds=True, count=64),
        # one decoded token behind a very long context in 32 bits, 96 of up to 4,096 pages of 32
        _case("picked token f32", "picked", "f32", 16, 4, 64, 64, 32, 1, 1, 131000, bounds=True, count=96),
    ]


MOST_CACHE = 64 * 8192 * 8 * 128          # features of the largest listed cache
MOST_PAIRS = 32 * 128 * 2048 * 1024       # features of queries x keys that they see, of the largest listed prompt


def _size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "picked"))
    dim = rng.choice((64, 64, 128, 128, 128, 192, 256))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 7, 8))
    while heads * dim > 4096:
        heads -= kv_heads
    case = {"op": op, "dtype": rng.choice(("bf16", "bf16", "f32")), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "group": rng.choice([g for g in (32, 64, 128) if dim % g == 0]), "window": 0, "lead": 0,
            "bounds": False, "rotary": dim, "neighbours": False, "count": 0}
    if op == "append":
        case["page"] = rng.choice((8, 16, 16, 24, 32, 64))
        case["requests"] = _size(rng, 1, 64)
        case["new"] = _size(rng, 1, max(1, 2048 // case["requests"]))
        case["held"] = rng.choice((0, _size(rng, 1, 8000)))
        case["rotary"] = rng.choice((dim, dim, dim // 2))
        case["neighbours"] = rng.random() < 0.3
        case["bounds"] = rng.random() < 0.3
        return case
    if op == "picked":
        case["page"] = rng.choice((16, 32, 64))
        case["requests"] = _size(rng, 1, 32)
        case["new"] = 1
        most = min(131072, MOST_CACHE // (2 * case["requests"] * kv_heads * dim))
        case["held"] = _size(rng, min(256, most), most) - 1
        case["bounds"] = True
        case["count"] = _size(rng, 4, 128)
        return case
    case["page"] = rng.choice((8, 16, 16, 24, 32, 64))
    if rng.random() < 0.6:                 # decoded tokens
        case["requests"], case["new"] = _size(rng, 1, 64), 1
    else:                                  # portions, single tokens among them
        case["requests"] = _size(rng, 1, 8)
        case["new"] = _size(rng, 2, 2048)
        case["lead"] = rng.randrange(0, case["requests"])
    most = min(131072, MOST_CACHE // (2 * case["requests"] * kv_heads * dim),
               MOST_PAIRS // (heads * dim * case["new"] * case["requests"]))
    if most <= case["new"]:
        case["new"] = max(1, min(case["new"], int(math.sqrt(MOST_PAIRS / (heads * dim * case["requests"])))))
        case["held"] = 0
    else:
        case["held"] = rng.choice((0, 1, 1, 1)) * (_size(rng, 1, most - case["new"] + 1) - 1)
    case["window"] = rng.choice((0, 0, 0, _size(rng, 16, 4096)))
    return case


# ---------------------------------------------------------------------------
# a step's requests
# ---------------------------------------------------------------------------

def _requests(case):
    """(held before the step, new in it) of every request: the first of the longest as long as the case says, the
    others down to half of that; `lead` requests at the head bring one token."""
    out = []
    for i in range(case["requests"]):
        less = (5 * i) % 8
        held = case["held"] - case["held"] * less // 16
        new = 1 if i < case["lead"] else case["new"] - case["new"] * (less if i > case["lead"] else 0) // 16
        out.append((held, max(1, new)))
    return out


def _rows(case):
    return sum(n for _, n in _requests(case))


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    requests, page = _requests(case), case["page"]
    heads, kv_heads, dim, groups = case["heads"], case["kv_heads"], case["dim"], case["dim"] // case["group"]
    state = dict(case)
    rows = sum(n for _, n in requests)
    state["new_tokens"], state["held_tokens"] = [n for _, n in requests], [h for h, _ in requests]
    state["positions"] = _ints([h + i for h, n in requests for i in range(n)])
    state["row_request"] = _ints([r for r, (_, n) in enumerate(requests) for _ in range(n)])
    starts = [0]
    for _, n in requests:
        starts.append(starts[-1] + n)
    state["row_start"] = _ints(starts)
    state["first_pos"] = _ints(state["held_tokens"])
    # every request's pages, scattered over the pool (appending reaches no page before a step's first, so that
    # those lie in one page that nobody writes)
    stride = max(-(-(h + n) // page) for h, n in requests)
    firsts = [h // page if case["op"] == "append" else 0 for h, _ in requests]
    counts = [-(-(h + n) // page) - f for (h, n), f in zip(requests, firsts)]
    pages = sum(counts) + 1
    scattered = torch.randperm(pages - 1, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for f, n in zip(firsts, counts):
        table.append([pages - 1] * f + scattered[at:at + n] + [pages - 1] * (stride - f - n))
        at += n
    state["table"] = _ints(table)
    # what is in the pool: codes of a bell's shape, groups of unlike sizes and places
    codes = torch.empty(2, pages, kv_heads, page, dim // 2, dtype=torch.uint8, device=DEV)
    for i in range(2):
        for p in range(0, pages, 4096):
            n = min(4096, pages - p)
            both = (_normal(gen, n, kv_heads, page, dim // 2, 2) * 2.9 + 7.5).round().clamp(0, 15).to(torch.uint8)
            codes[i, p:p + n] = both[..., 0] | (both[..., 1] << 4)
    step = 0.34 * torch.exp(0.2 * _normal(gen, 2, pages, kv_heads, page, groups))
    low = step * (-7.5 + 0.5 * _normal(gen, 2, pages, kv_heads, page, groups))
    state["codes"], state["scales"] = codes, torch.stack((step, low), dim=-1).to(torch.bfloat16)
    if case["bounds"]:
        state["bounds"] = torch.zeros(pages, kv_heads, 2, dim, dtype=torch.int8, device=DEV)
        state["bound_scales"] = torch.zeros(pages, kv_heads, device=DEV)
    dtype = FLOATS[case["dtype"]]
    if case["op"] == "append":
        # keys have a few features far larger than the others
        size = torch.exp(0.6 * _normal(gen, heads + 2 * kv_heads, dim))
        size[heads + kv_heads:] = 1.0
        state["qkv"] = (_normal(gen, rows, heads + 2 * kv_heads, dim) * size).view(rows, -1).to(dtype)
        half = case["rotary"] // 2
        angles = torch.outer(torch.arange(max(h + n for h, n in requests), dtype=torch.float64),
                             THETA ** (-torch.arange(half, dtype=torch.float64) / half))
        state["cos"], state["sin"] = angles.cos().float().to(DEV), angles.sin().float().to(DEV)
        state["q"] = torch.empty(rows, heads * dim, dtype=dtype, device=DEV)
        return state
    state["q"] = (1.2 * _normal(gen, rows, heads * dim)).to(dtype)
    state["scale"] = dim ** -0.5
    state["out"] = torch.empty(rows, heads * dim, dtype=dtype, device=DEV)
    if case["op"] == "picked":
        state["picks"] = torch.empty(rows, kv_heads, case["count"], dtype=torch.int32, device=DEV)
        for p in range(0, pages, 1024):
            values = _values(codes[0, p:p + 1024], state["scales"][0, p:p + 1024], case["group"])
            state["bounds"][p:p + 1024], state["bound_scales"][p:p + 1024] = _bounds(values, None)
    return state


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _features(dim):
    """For every feature its place among a row's groups of four bits."""
    word = torch.arange(dim // 8, device=DEV)
    g, w = word // (dim // 64), word % (dim // 64)
    feature = 64 * w[:, None] + 8 * torch.tensor(ORDER, device=DEV) + g[:, None]
    return torch.argsort(feature.reshape(-1))


def _values(codes, scales, group):
    """float32 rows [..., dim] that codes [..., dim / 2] and scales [..., dim / group, 2] stand for."""
    dim = 2 * codes.shape[-1]
    four = torch.stack((codes & 15, codes >> 4), dim=-1).view(*codes.shape[:-1], dim)
    four = four.index_select(-1, _features(dim)).float().view(*codes.shape[:-1], dim // group, group)
    pair = scales.float()
    return (four * pair[..., :1] + pair[..., 1:]).view(*codes.shape[:-1], dim)


def _bounds(values, held):
    """Bounds of pages [pages, kv heads, page tokens, dim] of which the first `held` tokens count (None: all)."""
    hi, lo = values, values
    if held is not None:
        there = torch.arange(values.shape[2], device=DEV) < held[:, None]
        hi = torch.where(there[:, None, :, None], values, -math.inf)
        lo = torch.where(there[:, None, :, None], values, math.inf)
    both = torch.stack((hi.amax(dim=2), lo.amin(dim=2)), dim=2)
    scale = both.abs().amax(dim=(2, 3)) * (1.0 / 127.0)
    inverse = torch.where(scale > 0, torch.reciprocal(scale), 0.0)
    return torch.round(both * inverse[..., None, None]).clamp(-127, 127).to(torch.int8), scale


def _rounded_down(x):
    """bfloat16 at or below x."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    return torch.where((bits < 0) & (bits != cut), cut + 65536, cut).view(torch.float32)


def _held(x, group):
    """What rows x [..., dim] come to in 4 bits."""
    parts = x.view(*x.shape[:-1], -1, group)
    low = _rounded_down(parts.amin(dim=-1, keepdim=True))
    step = ((parts.amax(dim=-1, keepdim=True) - low) * (1.0 / 15.0)).to(torch.bfloat16).float()
    step = torch.where(step < LEAST_STEP, 0.0, step)
    inverse = torch.where(step > 0, torch.reciprocal(step), 0.0)
    code = torch.round((parts - low) * inverse).clamp(0, 15)
    return (code * step + low).view(x.shape)


def _turned(x, cos, sin, rotary, neighbours):
    """Rows x [T, heads, dim] with their first `rotary` features turned; cos, sin [T, rotary / 2]."""
    cos, sin = cos[:, None], sin[:, None]
    turn = x[..., :rotary]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if neighbours else turn.chunk(2, dim=-1)
    pair = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.stack(pair, dim=-1).flatten(-2) if neighbours else torch.cat(pair, dim=-1)
    return torch.cat((turned, x[..., rotary:]), dim=-1)


def _plain_append(state):
    heads, kv_heads, dim, page = state["heads"], state["kv_heads"], state["dim"], state["page"]
    positions, dtype = state["positions"].long(), FLOATS[state["dtype"]]
    rows = state["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    cos, sin = state["cos"][positions], state["sin"][positions]
    turned = _turned(rows[:, :heads + kv_heads], cos, sin, state["rotary"], state["neighbours"])
    where = state["table"][state["row_request"].long(), positions // page].long()
    k = _values(state["codes"][0], state["scales"][0], state["group"])
    v = _values(state["codes"][1], state["scales"][1], state["group"])
    k[where, :, positions % page] = _held(turned[:, heads:].contiguous(), state["group"])
    v[where, :, positions % page] = _held(rows[:, heads + kv_heads:].contiguous(), state["group"])
    out = [turned[:, :heads].reshape(rows.shape[0], -1).to(dtype), k.to(dtype), v.to(dtype)]
    if state["bounds_kept"]:
        held = torch.zeros(k.shape[0], dtype=torch.int64, device=DEV)
        held.scatter_reduce_(0, where, positions % page + 1, reduce="amax")
        bounds, scale = _bounds(k, held.clamp_min(1))
        written = held > 0
        bounds = torch.where(written[:, None, None, None], bounds, state["bounds"]).float()
        out.append(bounds * torch.where(written[:, None], scale, state["bound_scales"])[..., None, None])
    return out


def _plain_scores(state):
    """The picking's scores [T, kv heads, pages of a table row], and each row's own page."""
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    q = state["q"].float().view(-1, heads, dim)
    scale = q.abs().amax(dim=-1) * (1.0 / 127.0)
    inverse = torch.where(scale > 0, torch.reciprocal(scale), 0.0)
    q8 = torch.round(q * inverse[..., None]).clamp(-127, 127).view(-1, kv_heads, heads // kv_heads, dim)
    table = state["table"][state["row_request"].long()].long()
    both = state["bounds"].float()[table]                      # [T, pages, kv heads, 2, dim]
    # (whole numbers below 2^24: every sum is exact)
    dots = (torch.einsum("thrd,tphd->thrp", q8.clamp_min(0), both[:, :, :, 0])
            + torch.einsum("thrd,tphd->thrp", q8.clamp_max(0), both[:, :, :, 1]))
    size = scale.view(-1, kv_heads, heads // kv_heads, 1) * state["bound_scales"][table].transpose(1, 2)[:, :, None]
    return (dots * size).amax(dim=2), state["positions"].long() // state["page"]


FIRST, LAST = 1, 2


def _plain_picks(state):
    score, own_page = _plain_scores(state)
    count, pages = state["count"], score.shape[-1]
    index = torch.arange(pages, device=DEV)
    always = (index < FIRST) | (index > own_page[:, None] - LAST)
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where((index > own_page[:, None])[:, None], -math.inf, score)
    # (a stable sort keeps the lowest index first among equals)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :count]
    best = torch.where(best > own_page[:, None, None], pages, best)
    if pages < count:
        best = torch.nn.functional.pad(best, (0, count - pages), value=pages)
    best = torch.sort(best, dim=-1).values
    return torch.where(best == pages, -1, best).to(torch.int32)


def _plain_attention(state, seen_pages=None):
    """All requests at once, behind padding; `seen_pages` [T, kv heads, pages]: the pages that a row sees."""
    heads, kv_heads, dim, page = state["heads"], state["kv_heads"], state["dim"], state["page"]
    new, requests = max(state["new_tokens"]), state["requests"]
    table = state["table"].long()
    keys = table.shape[1] * page
    k, v = (_values(state["codes"][i][table], state["scales"][i][table], state["group"]).transpose(1, 2)
            .reshape(requests, kv_heads, keys, dim) for i in range(2))
    row = state["row_start"][:-1, None].long() + torch.arange(new, device=DEV)
    there = row < state["row_start"][1:, None]
    row = row.clamp_max(state["q"].shape[0] - 1)
    q = state["q"].float()[row].view(requests, new, kv_heads, heads // kv_heads, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, -1, dim)
    logits = (q @ k.transpose(-1, -2)) * state["scale"]
    place = state["first_pos"][:, None] + torch.arange(new, device=DEV)          # [requests, new]
    key = torch.arange(keys, device=DEV)
    seen = key <= place[..., None]
    if state["window"]:
        seen &= key > place[..., None] - state["window"]
    seen = seen[:, None].expand(-1, kv_heads, -1, -1)
    if seen_pages is not None:
        seen = seen & seen_pages[row].permute(0, 2, 1, 3).repeat_interleave(page, dim=-1)
    logits = logits.view(requests, kv_heads, -1, new, keys).masked_fill_(~seen[:, :, None], -math.inf)
    logits -= logits.amax(dim=-1, keepdim=True)
    weights = logits.exp_()
    weights /= weights.sum(dim=-1, keepdim=True)
    out = weights.view(requests, kv_heads, -1, keys) @ v
    out = out.view(requests, kv_heads, heads // kv_heads, new, dim).permute(0, 3, 1, 2, 4).reshape(requests, new, -1)
    return out[there].to(FLOATS[state["dtype"]])


def run(state):
    op = state["op"]
    if own:
        from crucible_b200.ops import cache4
        kept = (state["bounds"], state["bound_scales"]) if torch.is_tensor(state["bounds"]) else (None, None)
        pages = cache4.Pages4(state["codes"], state["scales"], *kept)
        batch = cache4.Batch(state["positions"], state["row_request"], state["row_start"], state["first_pos"],
                             state["table"], state["new_tokens"], state["held_tokens"])
        if op == "append":
            cache4.rope_append4(state["qkv"], state["q"], state["heads"], state["cos"], state["sin"], batch, pages,
                                neighbours=state["neighbours"])
            out = [state["q"], *pages.values(FLOATS[state["dtype"]])]
            return out if kept[0] is None else [*out, pages.bound_values()]
        if op == "attend":
            cache4.attention4(state["q"], state["out"], state["heads"], state["scale"], batch, pages,
                              window=state["window"] or None)
            return state["out"]
        cache4.pick_pages4(state["q"], state["heads"], batch, pages, state["picks"], first=FIRST, last=LAST)
        cache4.attention4(state["q"], state["out"], state["heads"], state["scale"], batch, pages, picks=state["picks"])
        return [state["picks"], state["out"]]
    if op == "append":
        return _plain_append({**state, "bounds_kept": torch.is_tensor(state["bounds"])})
    if op == "attend":
        return _plain_attention(state)
    picks = _plain_picks(state)
    pages = state["table"].shape[1]
    seen = torch.zeros(*picks.shape[:2], pages + 1, dtype=torch.bool, device=DEV)
    seen.scatter_(2, torch.where(picks < 0, pages, picks).long(), True)
    return [picks, _plain_attention(state, seen[..., :pages])]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _visible(case, position):
    """Keys that a row at this position sees."""
    if case["op"] == "picked":
        full = min(position // case["page"] + 1, case["count"]) - 1
        return full * case["page"] + position % case["page"] + 1
    return min(position + 1, case["window"] or position + 1)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    heads, kv_heads, dim, rows = case["heads"], case["kv_heads"], case["dim"], _rows(case)
    token = kv_heads * (dim + 8 * (dim // case["group"]))           # bytes of a token's key and value
    if case["op"] == "append":
        pages = sum(-(-(h + n) // case["page"]) - h // case["page"] for h, n in _requests(case))
        moved = rows * (2 * heads + 2 * kv_heads) * dim * size + rows * (token + 4 * case["rotary"])
        moved += (pages + 1) * case["page"] * kv_heads * 2 * dim * size            # the pool as values
        if case["bounds"]:
            moved += pages * kv_heads * 2 * dim * 5
        return {"bytes": moved, "flops": rows * (heads + 2 * kv_heads) * dim * 6}
    pairs, keys, bounds = 0, 0, 0
    for held, new in _requests(case):
        pairs += sum(_visible(case, held + i) for i in range(new))
        keys += min(_visible(case, held + new - 1) + (new - 1 if case["window"] else 0), held + new)
        bounds += (held + new - 1) // case["page"] + 1
    moved = 2 * rows * heads * dim * size + keys * token
    flops = 4 * pairs * heads * dim
    if case["op"] == "picked":
        moved += bounds * kv_heads * (2 * dim + 4) + rows * kv_heads * case["count"] * 4
        flops += 4 * bounds * heads * dim
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_rows(state, which, page_ids):
    """float64 [kv heads, pages * page tokens, dim] of the pool's pages `page_ids`."""
    dim, group = state["dim"], state["group"]
    words = state["codes"][which][page_ids].view(torch.int32)              # [pages, kv heads, tokens, dim / 8]
    out = torch.empty(*words.shape[:-1], dim, dtype=torch.float64, device=DEV)
    per = dim // 64
    for n, k in enumerate(ORDER):
        four = torch.bitwise_and(torch.bitwise_right_shift(words, 4 * n), 15).double()
        for w in range(per):
            out[..., 64 * w + 8 * k:64 * w + 8 * k + 8] = four[..., w::per]
    pair = state["scales"][which][page_ids].double().repeat_interleave(group, dim=-2)
    out.mul_(pair[..., 0]).add_(pair[..., 1])
    return out.transpose(0, 1).reshape(words.shape[1], -1, dim)


def _once(x):
    """A result in 64 bits as float32 holds it.  (Sums, products and reciprocals of float32 numbers, taken in 64
    bits and then rounded, are those rounded once: 53 bits are more than twice 24 and two.)"""
    return x.float().double()


FIFTEENTH, OF_127 = (float(torch.tensor(1.0 / n, dtype=torch.float32)) for n in (15.0, 127.0))


def _exact_held(x, group):
    """Rows in 4 bits by the definition: the operations up to the code are float32's, the values exact."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], group):
        part = x[..., at:at + group]
        least, most = part.min(dim=-1, keepdim=True).values, part.max(dim=-1, keepdim=True).values
        low = least.to(torch.bfloat16)
        below = torch.nextafter(low, torch.full_like(low, -math.inf))
        low = torch.where(low.double() > least, below, low).double()
        step = _once(_once(most - low) * FIFTEENTH).to(torch.bfloat16).double()
        step = torch.where(step < LEAST_STEP, torch.zeros_like(step), step)
        inverse = _once(1.0 / step.clamp_min(1e-300))
        code = torch.where(step > 0, torch.round(_once(_once(part - low) * inverse)), torch.zeros_like(part))
        out[..., at:at + group] = torch.minimum(code.clamp_min(0), torch.full_like(code, 15)) * step + low
    return out


def _exact_append(state, case):
    heads, kv_heads, dim, page, rotary = (case[n] for n in ("heads", "kv_heads", "dim", "page", "rotary"))
    rows = state["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
    turn = rows[:, :heads + kv_heads].clone()
    coded = rows[:, heads:heads + kv_heads].clone()
    at = state["positions"].long()
    for i in range(rotary // 2):
        u, w = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + rotary // 2)
        c, s = state["cos"][at, i].double()[:, None], state["sin"][at, i].double()[:, None]
        a, b = rows[:, :heads + kv_heads, u], rows[:, :heads + kv_heads, w]
        turn[:, :, u] = a * c - b * s
        turn[:, :, w] = b * c + a * s
        a, b = a[:, heads:], b[:, heads:]
        coded[:, :, u] = _once(_once(a * c) - _once(b * s))
        coded[:, :, w] = _once(_once(a * s) + _once(b * c))
    everything = torch.arange(state["codes"].shape[1], device=DEV)
    k, v = (_exact_rows(state, i, everything).view(kv_heads, -1, page, dim).transpose(0, 1).contiguous() for i in range(2))
    new_k, new_v = _exact_held(coded, case["group"]), _exact_held(rows[:, heads + kv_heads:], case["group"])
    slot = state["table"][state["row_request"].long(), torch.div(at, page, rounding_mode="floor")].long()
    for h in range(kv_heads):
        k[slot, h, at % page] = new_k[:, h]
        v[slot, h, at % page] = new_v[:, h]
    out = [turn[:, :heads].reshape(rows.shape[0], -1), k, v]
    if case["bounds"]:
        held = {}
        for p, n in zip(slot.tolist(), (at % page + 1).tolist()):
            held[p] = max(held.get(p, 0), n)
        bounds = state["bounds"].double() * state["bound_scales"].double()[..., None, None]
        for p, n in held.items():
            hi, lo = k[p, :, :n].max(dim=1).values, k[p, :, :n].min(dim=1).values
            both = _once(torch.stack((hi, lo), dim=1))
            unit = _once(both.abs().flatten(1).max(dim=1).values * OF_127)[:, None, None]
            bounds[p] = torch.round(_once(both * _once(1.0 / unit))) * unit
        out.append(bounds)
    return out


def _exact_picks(state, case):
    """The picking by its definition: whole numbers, and float32 scores of them."""
    heads, kv_heads, dim, count = case["heads"], case["kv_heads"], case["dim"], case["count"]
    rep = heads // kv_heads
    out = torch.full((state["q"].shape[0], kv_heads, count), -1, dtype=torch.int32, device=DEV)
    for t, (r, p) in enumerate(zip(state["row_request"].tolist(), state["positions"].tolist())):
        last = p // case["page"]
        ids = state["table"][r, :last + 1].long()
        for h in range(kv_heads):
            most, least = state["bounds"][ids, h, 0].double(), state["bounds"][ids, h, 1].double()
            best = torch.full((last + 1,), -math.inf, device=DEV)
            for i in range(h * rep, (h + 1) * rep):
                q = state["q"][t, i * dim:(i + 1) * dim].float()
                unit = q.abs().max() * (1.0 / 127.0)
                q8 = torch.round(q * torch.reciprocal(unit)).double()
                dot = torch.maximum(q8 * most, q8 * least).sum(dim=1).float()
                best = torch.maximum(best, dot * (unit * state["bound_scales"][ids, h]))
            best[:FIRST] = math.inf
            best[max(0, last - LAST + 1):] = math.inf
            rank = torch.argsort(best, descending=True, stable=True)[:count]
            out[t, h, :rank.numel()] = torch.sort(rank).values.to(torch.int32)
    return out


def _exact_attention(state, case, picks=None):
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rep, row = heads // kv_heads, 0
    out = torch.zeros(state["q"].shape[0], heads * dim, dtype=torch.float64, device=DEV)
    for r, (held, new) in enumerate(_requests(case)):
        ids = state["table"][r, :-(-(held + new) // page)].long()
        k, v = _exact_rows(state, 0, ids), _exact_rows(state, 1, ids)
        key = torch.arange(k.shape[1], device=DEV)
        for at in range(0, new, 256):
            n = min(256, new - at)
            place = held + at + torch.arange(n, device=DEV)[:, None]
            hidden = key > place
            if case["window"]:
                hidden = hidden | (key <= place - case["window"])
            for h in range(heads):
                unseen = hidden
                if picks is not None:
                    listed_pages = picks[row + at, h // rep]
                    seen = torch.zeros(ids.numel(), dtype=torch.bool, device=DEV)
                    seen[listed_pages[listed_pages >= 0].long()] = True
                    unseen = hidden | ~seen.repeat_interleave(page)
                q = state["q"][row + at:row + at + n, h * dim:(h + 1) * dim].double()
                logits = torch.where(unseen, -math.inf, torch.mm(q, k[h // rep].t()) * state["scale"])
                weights = torch.softmax(logits, dim=1)
                out[row + at:row + at + n, h * dim:(h + 1) * dim] = torch.mm(weights, v[h // rep])
        row += new
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(state, case)
    if case["op"] == "attend":
        return _exact_attention(state, case)
    picks = _exact_picks(state, case)
    return [picks, _exact_attention(state, case, picks)]
