"""What the operators over the cache in 4 bits are held against: the format and the operators by their definitions, in
64 bits (and, up to the codes, in float32 one operation at a time), a row at a time."""
from __future__ import annotations

import math

import torch

ORDER = (0, 1, 4, 5, 2, 3, 6, 7)
LEAST_STEP = 1e-30


def once(x):
    """float32 of a result in 64 bits: what a float32 operation gives."""
    return x.float().double()


FIFTEENTH = float(torch.tensor(1.0 / 15.0, dtype=torch.float32))
OF_127 = float(torch.tensor(1.0 / 127.0, dtype=torch.float32))


def bf16_below(x):
    y = x.to(torch.bfloat16)
    return torch.where(y.double() > x, torch.nextafter(y, torch.full_like(y, -math.inf)), y)


def coded(x, group):
    """x float64 [..., D] of float32 numbers -> codes int64 [..., D], step, low bfloat16 [..., D / group]."""
    parts = x.unflatten(-1, (-1, group))
    low = bf16_below(parts.amin(dim=-1))
    step = once(once(parts.amax(dim=-1) - low.double()) * FIFTEENTH).to(torch.bfloat16)
    step = torch.where(step.double() < LEAST_STEP, torch.zeros_like(step), step)
    inverse = torch.where(step > 0, once(1.0 / step.double().clamp_min(1e-300)), 0.0)
    code = torch.round(once(once(parts - low.double()[..., None]) * inverse[..., None])).clamp(0, 15)
    return code.long().flatten(-2), step, low


def packed(codes):
    """int64 codes [..., D] -> uint8 [..., D / 2] as they lie in memory."""
    dim = codes.shape[-1]
    words = torch.zeros(*codes.shape[:-1], dim // 8, dtype=torch.int64, device=codes.device)
    for f in range(dim):
        w, k, g = f // 64, f % 64 // 8, f % 8
        words[..., dim // 64 * g + w] |= codes[..., f] << (4 * ORDER.index(k))
    return torch.stack([(words >> (8 * i)) & 255 for i in range(4)], dim=-1).flatten(-2).to(torch.uint8)


def unpacked(codes):
    dim = 2 * codes.shape[-1]
    bytes4 = codes.long().unflatten(-1, (-1, 4))
    words = sum(bytes4[..., i] << (8 * i) for i in range(4))
    out = torch.empty(*codes.shape[:-1], dim, dtype=torch.int64, device=codes.device)
    for f in range(dim):
        w, k, g = f // 64, f % 64 // 8, f % 8
        out[..., f] = (words[..., dim // 64 * g + w] >> (4 * ORDER.index(k))) & 15
    return out


def values(codes, scales):
    """float64 rows that packed codes [..., D / 2] and scales [..., D / group, 2] stand for."""
    four = unpacked(codes).double()
    group = four.shape[-1] // scales.shape[-2]
    pair = scales.double().repeat_interleave(group, dim=-2)
    return four * pair[..., 0] + pair[..., 1]


def turned(x, cos, sin, neighbours):
    """Rows x float64 [T, heads, D], angles' cos and sin [T, r / 2]: rotated in float32, one operation at a time."""
    out = x.clone()
    half = cos.shape[-1]
    for i in range(half):
        u, w = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        a, b, c, s = x[..., u], x[..., w], cos[:, None, i].double(), sin[:, None, i].double()
        out[..., u] = once(once(a * c) - once(b * s))
        out[..., w] = once(once(a * s) + once(b * c))
    return out


def tables(positions, half, device, theta=10000.0):
    angles = torch.outer(torch.arange(positions, dtype=torch.float64),
                         theta ** (-torch.arange(half, dtype=torch.float64) / max(1, half)))
    return angles.cos().float().to(device), angles.sin().float().to(device)


class Case:
    """Requests (held, new) over scattered pages of random content; one more page than they need, which no table names."""

    def __init__(self, requests, dim=64, kv_heads=2, n_rep=3, page=16, group=32, dtype=torch.bfloat16, seed=0, bounds=False,
                 device="cuda:0", size=1.0):
        from crucible_b200.ops import cache4
        gen = torch.Generator(device=device).manual_seed(seed)
        self.gen, self.device, self.requests, self.dim, self.kv_heads = gen, device, requests, dim, kv_heads
        self.heads, self.page, self.group, self.dtype = kv_heads * n_rep, page, group, dtype
        counts = [-(-(h + n) // page) for h, n in requests]
        self.stride = max(counts)
        self.n_pages = sum(counts) + 1
        order = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed + 1)).tolist()
        self.free = order.pop()
        table = []
        for n in counts:
            table.append([order.pop() for _ in range(n)] + [self.free] * (self.stride - n))
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.table = ints(table)
        self.positions = ints([h + i for h, n in requests for i in range(n)])
        self.row_request = ints([r for r, (_, n) in enumerate(requests) for _ in range(n)])
        starts = [0]
        for _, n in requests:
            starts.append(starts[-1] + n)
        self.rows = starts[-1]
        self.row_start, self.first_pos = ints(starts), ints([h for h, _ in requests])
        shape = (2, self.n_pages, kv_heads, page)
        codes = torch.randint(0, 256, (*shape, dim // 2), generator=gen, device=device, dtype=torch.uint8)
        step = 0.3 * torch.exp(0.3 * torch.randn(*shape, dim // group, generator=gen, device=device)) * size
        low = step * (-7.5 + torch.randn(*shape, dim // group, generator=gen, device=device))
        scales = torch.stack((step, low), dim=-1).to(torch.bfloat16)
        self.pages = cache4.Pages4(codes, scales, *(() if not bounds else (
            torch.zeros(self.n_pages, kv_heads, 2, dim, dtype=torch.int8, device=device),
            torch.zeros(self.n_pages, kv_heads, device=device))))
        self.batch = self.make_batch()

    def make_batch(self, **more):
        from crucible_b200.ops import cache4
        return cache4.Batch(self.positions, self.row_request, self.row_start, self.first_pos, self.table,
                            [n for _, n in self.requests], [h for h, _ in self.requests], **more)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=self.device)

    def queries(self, size=1.0):
        return (size * self.normal(self.rows, self.heads * self.dim)).to(self.dtype)

    def contents(self):
        """float64 [2, pages, kv heads, page tokens, D]."""
        return values(self.pages.codes, self.pages.scales)

    def attention(self, q, scale, window=None, picks=None, spread=None):
        """(results, the largest magnitude of a value that a row sees) in float64, each [rows, heads * dim].  `spread`, a list:
        also gets scale * max_j sum_f |q_f| |k_jf| of every row and head."""
        everything = self.contents()
        rep = self.heads // self.kv_heads
        out = torch.zeros(self.rows, self.heads, self.dim, dtype=torch.float64, device=self.device)
        most = torch.zeros(self.rows, self.heads, 1, dtype=torch.float64, device=self.device)
        terms = torch.zeros(self.rows, self.heads, 1, dtype=torch.float64, device=self.device)
        row = 0
        table, positions = self.table.tolist(), self.positions.tolist()
        for r, (_, new) in enumerate(self.requests):
            for i in range(row, row + new):
                pos = positions[i]
                for h in range(self.kv_heads):
                    lo = 0 if window is None else max(0, pos - window + 1)
                    keys = range(lo, pos + 1)
                    if picks is not None:
                        own = set(picks[i, h].tolist())
                        keys = [j for j in keys if j // self.page in own]
                    keys = [j for j in keys if j // self.page < self.stride and 0 <= table[r][j // self.page] < self.n_pages]
                    if not keys:
                        continue
                    at = torch.tensor(keys, device=self.device)
                    where = torch.tensor([table[r][j // self.page] for j in keys], device=self.device)
                    k, v = everything[0][where, h, at % self.page], everything[1][where, h, at % self.page]
                    heads = q[i].double().view(self.heads, self.dim)[h * rep:(h + 1) * rep]
                    weights = torch.softmax(heads @ k.t() * scale, dim=-1)
                    out[i, h * rep:(h + 1) * rep] = weights @ v
                    most[i, h * rep:(h + 1) * rep] = v.abs().amax()
                    terms[i, h * rep:(h + 1) * rep] = (heads.abs() @ k.abs().t()).amax(dim=1, keepdim=True) * scale
            row += new
        if spread is not None:
            spread.append(terms.expand(-1, -1, self.dim).flatten(1))
        return out.flatten(1), most.expand(-1, -1, self.dim).flatten(1)


def assert_attention(got, want, most, dtype):
    """bfloat16: the result's rounding, and p step in float16 (half a step is 2^-12 of at most 2 max|v| 16/15), sums of
    products of subnormals that the tensor cores cut at 2^-14 of the largest, scores likewise (2^-14 of a score's
    terms moves p by less than 2^-9): 2^-9 max|v| in all.  float32: scores of up to 32 (in log2) are rounded at 2^-20 and
    move p by as much, twice (its sum too); two float16 parts are off by 2^-22: 2^-17 max|v| in all."""
    off, more = (2.0 ** -8, 2.0 ** -9) if dtype == torch.bfloat16 else (2.0 ** -24, 2.0 ** -17)
    assert torch.isfinite(got.float()).all()
    worst = ((got.double() - want).abs() - (off * want.abs() + more * most)).max()
    assert float(worst) <= 0.0, f"over by {float(worst)}"


def assert_attention_laid_out(got, want, most, terms):
    """bfloat16 portions whose keys and values are laid out in float16: values are off by 2^-11 of themselves, p by 2^-11 (its sum
    is float32's), keys and queries by 2^-11 and 2^-28, so that a score is off by d = 2^-11 scale sum |q| |k| at most
    and a weight by a factor of e^(2 d); on top the result's rounding, and 2^-10 for the tensor cores' and the sum's float32."""
    moved = torch.expm1(2 * 1.001 * 2.0 ** -11 * terms)
    worst = ((got.double() - want).abs() - (2.0 ** -8 * want.abs() + (2 * 2.0 ** -11 + 2.0 ** -10 + moved) * most)).max()
    assert torch.isfinite(got.float()).all() and float(worst) <= 0.0, f"over by {float(worst)}"
