"""Plain 64-bit forms of the quantised operators, and what their kernels' rounding may come to."""
import torch

E4M3 = torch.float8_e4m3fn
TOP, LEAST = 448.0, 1e-30


def step_of(v):
    """The distance of neighbouring e4m3 numbers around v (float64, at most 448)."""
    return torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(2.0 ** -6, TOP)).exponent - 4)


def check_rows8(q, scales, y, what=""):
    """q (e4m3) and scales against the float64 rows y.  A kernel takes y and its scale with at most 64
    roundings of 2^-24 each (sums of squares add up as a tree, its root halves them; the rest are a dozen
    products), and rounds once to e4m3, which is off by half a step at most; so is a number that those
    64 roundings took across the border of two."""
    near = 64 * 2.0 ** -24
    want = y.abs().amax(dim=1).clamp_min(LEAST) / TOP
    assert ((scales.double() - want).abs() <= near * want).all(), f"{what}: scales"
    v = y / want[:, None]
    off = (q.double() - v).abs() - (0.5 * step_of(v) + 2 * near * v.abs())
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} numbers, the worst by {float(off.max())}"


def exact_norm(x, delta, gain, eps):
    total = x.double() + (delta.double() if delta is not None else 0.0)
    return total, total / torch.sqrt(total.pow(2).mean(dim=1, keepdim=True) + eps) * gain.double()


def exact_glu(both, limit, alpha=1.0, offset=0.0):
    g, u = both.double().chunk(2, dim=1)
    if limit is None:
        return g * torch.sigmoid(g) * u
    return g.clamp(max=limit) * torch.sigmoid(alpha * g.clamp(max=limit)) * (u.clamp(-limit, limit) + offset)


def dense8(w):
    return w.values.double() * w.scales.double()[:, None]


def dense4(w):
    n, k = w.shape
    out = torch.empty(n, k, dtype=torch.float64, device=w.codes.device)
    for i in range(8):
        out[:, i::8] = (((w.codes >> (4 * (i // 2) + 16 * (i % 2))) & 15) - 8).double()
    return out * w.group_scales.double().repeat_interleave(w.group, dim=1) * w.scales.double()[:, None]


def check_product(out, rows, weights, add, passes=1, what=""):
    """`out` against float64 rows . weights^T (+ add).  The tensor cores add 16 products (or 32) and the sum
    so far at a time, which may be cut instead of rounded: a step of 2^-23 each, relative to the sum
    of the magnitudes; `passes`: bfloat16 parts of a float32 row.  32 more for the sums of warps or blocks, the
    scales and the addition, and the rounding to the output's type."""
    want = rows @ weights.t()
    size = rows.abs() @ weights.abs().t()
    if add is not None:
        want, size = want + add.double(), size + add.double().abs()
    k = rows.shape[1]
    bound = (passes * -(-k // 16) + 32) * 2.0 ** -23 * size
    bound += (want.abs() + bound) * (torch.finfo(out.dtype).eps / 2)
    off = (out.double() - want).abs() - bound
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} of {off.numel()}, the worst by {float(off.max())}"


def random_weights4(n, k, group, device, gen):
    from crucible_b200.ops import quantized
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int64, generator=gen, device=device).to(torch.int32)
    # every scale that e4m3 has, negative ones and zeros too, but NaN
    scale = torch.randint(0, 256, (n, k // group), generator=gen, device=device).to(torch.uint8)
    scale[(scale & 127) == 127] = 0
    return quantized.Weights4(codes, scale.view(E4M3), torch.rand(n, generator=gen, device=device) + 0.5)


def random_weights8(n, k, device, gen):
    from crucible_b200.ops import quantized
    values = torch.randint(0, 256, (n, k), generator=gen, device=device).to(torch.uint8)
    values[(values & 127) == 127] = 0
    return quantized.Weights8(values.view(E4M3), torch.rand(n, generator=gen, device=device) + 0.5)


def random_rows8(rows, k, device, gen):
    from crucible_b200.ops import quantized
    q = quantized.new_rows8(rows, k, device)
    v = torch.randint(0, 256, (rows, k), generator=gen, device=device).to(torch.uint8)
    v[(v & 127) == 127] = 0
    q.view(torch.uint8).copy_(v)
    return q, torch.rand(rows, generator=gen, device=device) + 0.5
