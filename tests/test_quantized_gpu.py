"""The quantised operators' kernels against plain 64-bit forms."""
import pytest
import torch

from crucible_b200.ops import KernelError, quantized
from quantized_cases import (E4M3, LEAST, TOP, check_product, check_rows8, dense4, dense8, exact_glu, exact_norm,
                             random_rows8, random_weights4, random_weights8)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(seed=11):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _framed(rows, width, dtype, left, right, fill):
    """Rows inside a larger buffer, so that a write beside them shows: (the rows, the buffer's frame)."""
    buf = torch.full((rows + 2, left + width + right), fill, device=DEV).to(dtype)
    return buf[1:rows + 1, left:left + width], buf


def _frame_kept(inner, buf, left, fill):
    rows, width = inner.shape
    frame = buf.float().clone()
    frame[1:rows + 1, left:left + width] = fill
    assert (frame == fill).all(), "something beside the rows was written"


WIDTHS = [1, 3, 4, 63, 64, 100, 128, 129, 256, 511, 512, 513, 700, 768, 1000, 2048, 4096, 5000, 14336, 16384, 16388, 32768]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("delta", ["none", "f32", "bf16"])
def test_add_rmsnorm8(width, delta):
    gen = _gen(width)
    for rows, left, right in ((1, 0, 0), (5, 4, 4), (6, 1, 2)):
        wide = _randn(gen, rows, width + 8) * torch.exp(_randn(gen, rows, 1))
        x = wide[:, left:left + width]
        d = (0.5 * _randn(gen, rows, width)).to(DTYPES[delta]) if delta != "none" else None
        gain = 1 + 0.2 * _randn(gen, width)
        total, y = exact_norm(x, d, gain, 1e-5)
        q, frame = _framed(rows, width, E4M3, left, right, 3.0)
        s = torch.empty(rows, device=DEV)
        sums, sum_frame = _framed(rows, width, torch.float32, left, right, 3.0)
        before = x.clone()
        quantized.add_rmsnorm8(x, d, gain, 1e-5, q, s, sum_out=sums)
        check_rows8(q, s, y, f"{rows} rows")
        assert torch.equal(x, before)
        assert ((sums.double() - total).abs() <= total.abs() * 2.0 ** -24).all()
        _frame_kept(q, frame, left, 3.0)
        _frame_kept(sums, sum_frame, left, 3.0)
        # in place: the same numbers, bit for bit
        q2, s2 = quantized.new_rows8(rows, width, DEV), torch.empty(rows, device=DEV)
        quantized.add_rmsnorm8(x, d, gain, 1e-5, q2, s2)
        assert torch.equal(x, sums if d is not None else before)
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s, s2)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pair", [(None, 1.0, 0.0), (2.0, 1.702, 1.0)])
def test_glu8(width, dtype, pair):
    gen = _gen(width)
    for rows, left, right in ((1, 0, 0), (5, 4, 4), (6, 1, 2)):
        both = (2 * _randn(gen, rows, 2 * width + 8)).to(DTYPES[dtype])[:, left:left + 2 * width]
        q, frame = _framed(rows, width, E4M3, left, right, 3.0)
        s = torch.empty(rows, device=DEV)
        quantized.glu8(both, q, s, *pair)
        check_rows8(q, s, exact_glu(both, *pair), f"{rows} rows")
        _frame_kept(q, frame, left, 3.0)


@pytest.mark.parametrize("dtype,width", [("bf16", 8192), ("bf16", 8200), ("bf16", 14336), ("bf16", 14344), ("bf16", 28800), ("bf16", 28808),
                                         ("bf16", 9001), ("f32", 4100), ("f32", 7168), ("f32", 7172), ("f32", 14400), ("f32", 14404)])
@pytest.mark.parametrize("rows", [1023, 1024, 1337])
def test_glu8_of_many_long_rows(dtype, width, rows):
    """Around the sizes from which rows come through shared memory, by blocks of either size, to which they do."""
    gen = _gen(width + rows)
    wide = (2 * _randn(gen, rows, 2 * width + 8)).to(DTYPES[dtype])
    both = wide[:, :2 * width]
    both[rows - 1, 5], both[7, width + 1] = float("nan"), float("inf")
    both[8] = 0.0
    for limit, alpha, offset in ((None, 1.0, 0.0), (2.0, 1.25, 0.75)):
        out, scales = quantized.new_rows8(rows, width, DEV), torch.full((rows + 1,), -1.0, device=DEV)
        quantized.glu8(both, out, scales[:rows], limit, alpha, offset)
        y = exact_glu(both, limit, alpha, offset)
        fine = torch.isfinite(y).all(dim=1)
        assert int(fine.sum()) == (rows - 2 if limit is None else rows - 1) and scales[rows] == -1.0
        check_rows8(out[fine], scales[:rows][fine], y[fine], f"{dtype} {rows} x {width} {limit}")
        assert not torch.isfinite(scales[:rows][~fine]).any()


@pytest.mark.parametrize("width", [5, 64, 768, 4096, 20000])
def test_rows8_of_zeros_and_of_what_is_no_number(width):
    nan, inf = float("nan"), float("inf")
    x = torch.ones(5, width, device=DEV)
    x[0] = 0.0
    x[1, width // 2] = nan
    x[2, width - 1] = inf
    x[3] *= 1e-25                      # the norm's eps holds it down: 1e-25 / sqrt(1e-5), above LEAST
    q, s = quantized.new_rows8(5, width, DEV), torch.empty(5, device=DEV)
    gain = torch.ones(width, device=DEV)
    quantized.add_rmsnorm8(x, None, gain, 1e-5, q, s)
    v = q.float()
    assert (v[0] == 0).all() and float(s[0]) == pytest.approx(LEAST / TOP, rel=1e-6)
    assert torch.isnan(s[1]) and torch.isnan(v[1]).all()
    assert torch.isnan(s[2]) and torch.isnan(v[2]).all()
    assert (v[3] == TOP).all() and (v[4] == TOP).all()
    assert float(s[4]) == pytest.approx(1 / TOP, rel=1e-5)
    both = torch.ones(3, 2 * width, device=DEV)
    both[0, :width] = 0.0
    both[1, width - 1] = nan
    both[2, width] = inf
    q, s = quantized.new_rows8(3, width, DEV), torch.empty(3, device=DEV)
    quantized.glu8(both, q, s)
    v = q.float()
    assert (v[0] == 0).all() and float(s[0]) == pytest.approx(LEAST / TOP, rel=1e-6)
    assert torch.isnan(s[1]) and torch.isnan(v[1]).all()
    # an infinity: the scale is one, the finite numbers vanish beside it, it itself is no number of e4m3
    assert torch.isinf(s[2]) and torch.isnan(v[2, 0]) and (v[2, 1:] == 0).all()


@pytest.mark.parametrize("pair", [(None, 1.0, 0.0), (7.0, 1.702, 1.0), (1e30, 1.0, 0.0)])
def test_glu8_far_from_zero(pair):
    """Gates whose exponential is nothing, or more than 32 bits hold."""
    g = torch.tensor([0.0, 1e-30, -1e-30, 20.0, -20.0, 60.0, -60.0, 87.0, -87.0, 100.0, -100.0, 1e6, -1e6, 3e38, -3e38, 0.5], device=DEV)
    rows = []
    for i in range(16):                                # each gate beside small ones, so that none of them hides it
        r = torch.full((16,), 0.25, device=DEV)
        r[i] = g[i]
        rows.append(torch.cat([r, torch.ones(16, device=DEV)]))
    both = torch.stack(rows)
    q, s = quantized.new_rows8(16, 16, DEV), torch.empty(16, device=DEV)
    quantized.glu8(both, q, s, *pair)
    check_rows8(q, s, exact_glu(both, *pair))


def test_rows8_refuse_what_no_block_holds():
    x, q, s = torch.zeros(1, 32769, device=DEV), quantized.new_rows8(1, 32769, DEV), torch.zeros(1, device=DEV)
    with pytest.raises(KernelError, match="32768"):
        quantized.add_rmsnorm8(x, None, torch.ones(32769, device=DEV), 1e-5, q, s)
    with pytest.raises(KernelError, match="32768"):
        quantized.glu8(torch.zeros(1, 2 * 32769, device=DEV), q, s)
    quantized.add_rmsnorm8(x[:0, :8], None, torch.ones(8, device=DEV), 1e-5, q[:0, :8], s[:0])     # no rows: nothing


ROWS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 128, 130, 257, 300]


def _check8(rows, n, k, out_dtype, add, seed=0):
    gen = _gen(seed + rows * 7919 + n * 31 + k)
    w = random_weights8(n, k, DEV, gen)
    q, s = random_rows8(rows, k, DEV, gen)
    out, frame = _framed(rows, n, out_dtype, 3, 2, 3.0)
    plus = 100 * _randn(gen, rows, n) if add else None
    quantized.linear8(q, s, w, out, add=plus)
    check_product(out, q.double() * s.double()[:, None], dense8(w), plus, what=f"{rows}x{n}x{k}")
    _frame_kept(out, frame, 3, 3.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_linear8_rows(rows, out):
    for n, k in ((1, 16), (5, 1), (16, 64), (17, 100), (100, 129), (127, 256), (129, 1000), (300, 513)):
        _check8(rows, n, k, DTYPES[out], rows % 2 == 0)


@pytest.mark.parametrize("n,k", [(6144, 4096), (4096, 14336), (1000, 16383), (5631, 1000), (40000, 128)])
def test_linear8_sizes(n, k):
    for rows in (1, 8, 33, 130):
        _check8(rows, n, k, torch.float32, True)


@pytest.mark.parametrize("rows,n,k", [(1024, 1280, 768), (2000, 4096, 2048), (4097, 300, 96), (700, 5631, 1000)])
def test_linear8_prompts(rows, n, k):
    _check8(rows, n, k, torch.bfloat16, False)
    _check8(rows, n, k, torch.float32, True)


@pytest.mark.parametrize("form", ["few", "tiles", "pairs"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 130, 100), (16, 257, 129), (17, 128, 128), (40, 255, 600), (129, 300, 1000),
                                      (250, 513, 256), (257, 700, 2049), (300, 256, 6000), (513, 40000, 64)])
def test_linear8_by_every_form(form, rows, n, k, monkeypatch):
    monkeypatch.setattr(quantized, "FORM", form)
    for out, add in ((torch.float32, True), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)):
        _check8(rows, n, k, out, add)


@pytest.mark.parametrize("form", ["few", "ring", "tiles", "pairs"])
@pytest.mark.parametrize("rows,n,k,group", [(1, 1, 32, 32), (3, 130, 96, 96), (16, 257, 160, 32), (17, 128, 256, 64),
                                            (40, 255, 608, 32), (129, 300, 1024, 128), (250, 513, 288, 96),
                                            (257, 700, 2080, 32), (300, 256, 6144, 6144), (513, 40000, 64, 64)])
def test_linear4_by_every_form(form, rows, n, k, group, monkeypatch):
    monkeypatch.setattr(quantized, "FORM", form)
    for dtype in (torch.bfloat16, torch.float32):
        for out, add in ((torch.float32, True), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)):
            _check4(rows, n, k, group, dtype, out, add)


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("n,k,group", [(1, 256, 32), (33, 256, 256), (64, 512, 64), (100, 1024, 32), (129, 1280, 160), (300, 1536, 96),
                                       (18944, 768, 128), (20000, 256, 64), (40000, 512, 32), (31, 4096, 2048)])
def test_linear4_by_the_ring(rows, n, k, group, monkeypatch):
    """Every number of groups, K of one stage and of several, scales that begin inside a segment."""
    monkeypatch.setattr(quantized, "FORM", "ring")
    _check4(rows, n, k, group, torch.bfloat16, torch.float32, True)
    _check4(rows, n, k, group, torch.bfloat16, torch.bfloat16, False)


@pytest.mark.parametrize("block", [(1, 8), (1, 4), (2, 4), (2, 2)])
@pytest.mark.parametrize("shares", [1, 2, 3, 4, 8])
def test_linear4_by_rings_that_share_k(block, shares, monkeypatch):
    monkeypatch.setattr(quantized, "_rule", lambda *sizes: ("ring", *block, shares))
    for rows, n, k, group in ((1, 33, 256, 32), (8, 100, 2304, 64), (9, 64, 4096, 4096), (20, 129, 1280, 160), (3, 31, 8448, 96)):
        _check4(rows, n, k, group, torch.bfloat16, torch.float32, True)
        _check4(rows, n, k, group, torch.bfloat16, torch.bfloat16, False)
    for rows, n, k, group in ((1, 33, 256, 32), (2, 100, 2304, 64), (3, 64, 4096, 4096), (5, 129, 1280, 160)):
        _check4(rows, n, k, group, torch.float32, torch.float32, True)
        _check4(rows, n, k, group, torch.float32, torch.bfloat16, False)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 6])
def test_few_float32_rows(rows):
    """Those that the ring takes as three rows each, and one more."""
    for n, k, group in ((1000, 768, 64), (2048, 8192, 128), (300, 4096, 32), (12000, 256, 256)):
        _check4(rows, n, k, group, torch.float32, torch.float32, rows % 2 == 0)


def test_six_float32_rows_are_too_many_for_the_ring(monkeypatch):
    monkeypatch.setattr(quantized, "_rule", lambda *sizes: ("ring", 1, 8, 1))
    gen = _gen()
    with pytest.raises(KernelError, match="sizes out of range"):
        quantized.linear4(_randn(gen, 6, 256), random_weights4(32, 256, 32, DEV, gen), torch.empty(6, 32, device=DEV))


@pytest.mark.parametrize("rows,n,k,group", [(1, 2048, 8192, 64), (8, 500, 14336, 128), (16, 1280, 4096, 64), (20, 512, 8192, 32)])
def test_linear4_of_few_features(rows, n, k, group):
    _check4(rows, n, k, group, torch.bfloat16, torch.float32, True)


def _check4(rows, n, k, group, dtype, out_dtype, add, seed=0):
    gen = _gen(seed + rows * 7919 + n * 31 + k)
    w = random_weights4(n, k, group, DEV, gen)
    a = (_randn(gen, rows, k) * torch.exp(2 * _randn(gen, rows, k))).to(dtype)
    out, frame = _framed(rows, n, out_dtype, 3, 2, 3.0)
    plus = 100 * _randn(gen, rows, n) if add else None
    quantized.linear4(a, w, out, add=plus)
    check_product(out, a.double(), dense4(w), plus, 3 if dtype == torch.float32 else 1, f"{rows}x{n}x{k}/{group}")
    _frame_kept(out, frame, 3, 3.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear4_rows(rows, dtype):
    for n, k, group in ((1, 32, 32), (5, 64, 64), (16, 96, 32), (17, 128, 128), (100, 160, 160), (127, 384, 96),
                        (129, 1024, 64), (300, 544, 32)):
        _check4(rows, n, k, group, DTYPES[dtype], torch.float32 if n % 2 else torch.bfloat16, rows % 2 == 0)


@pytest.mark.parametrize("n,k,group", [(28672, 4096, 64), (2048, 8192, 32), (4096, 14336, 128), (1000, 16384, 4096),
                                       (40000, 128, 32)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear4_sizes(n, k, group, dtype):
    for rows in (1, 8, 33, 130):
        _check4(rows, n, k, group, DTYPES[dtype], torch.float32, True)


@pytest.mark.parametrize("rows,n,k,group", [(1024, 1280, 768, 64), (2000, 4096, 2048, 128), (4097, 300, 96, 32),
                                            (700, 5631, 1024, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear4_prompts(rows, n, k, group, dtype):
    _check4(rows, n, k, group, DTYPES[dtype], torch.bfloat16, False)
    _check4(rows, n, k, group, DTYPES[dtype], torch.float32, True)


@pytest.mark.parametrize("rows", [128, 129, 300])
def test_float32_rows_a_slab_at_a_time(rows, monkeypatch):
    monkeypatch.setattr(quantized, "_SLAB", 128)
    _check4(rows, 200, 256, 64, torch.float32, torch.float32, True)
    _check4(rows, 200, 256, 64, torch.float32, torch.bfloat16, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear4_millions_of_rows(dtype):
    _check4(4_200_000, 3, 32, 32, DTYPES[dtype], torch.float32, False)


@pytest.mark.parametrize("rows", [1, 8, 40, 300])
def test_products_add_into_their_output(rows):
    gen = _gen(rows)
    w8, w4 = random_weights8(200, 256, DEV, gen), random_weights4(200, 256, 64, DEV, gen)
    q, s = random_rows8(rows, 256, DEV, gen)
    a = _randn(gen, rows, 256).bfloat16()
    before = 50 * _randn(gen, rows, 200)
    for call, exact, weights in ((lambda out: quantized.linear8(q, s, w8, out, add=out), q.double() * s.double()[:, None], dense8(w8)),
                                 (lambda out: quantized.linear4(a, w4, out, add=out), a.double(), dense4(w4))):
        out, apart = before.clone(), torch.empty_like(before)
        call(out)
        check_product(out, exact, weights, before)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_rows_of_any_stride_and_alignment(rows):
    """Rows that do not begin on 16 bytes, rows apart, one row of a strange stride."""
    gen = _gen(rows)
    for k, left in ((64, 0), (64, 1), (96, 3), (128, 8)):
        w8, w4 = random_weights8(70, k, DEV, gen), random_weights4(70, k, 32, DEV, gen)
        out = torch.empty(rows, 70, device=DEV)
        v = torch.randint(0, 120, (rows, k + 9), generator=gen, device=DEV).to(torch.uint8).view(E4M3)[:, left:left + k]
        s = torch.rand(2 * rows, generator=gen, device=DEV)[rows:]
        quantized.linear8(v, s, w8, out)
        check_product(out, v.double() * s.double()[:, None], dense8(w8), None)
        for dtype in (torch.float32, torch.bfloat16):
            a = _randn(gen, rows, k + 9).to(dtype)[:, left:left + k]
            quantized.linear4(a, w4, out)
            check_product(out, a.double(), dense4(w4), None, 3)
    odd = random_weights8(70, 50, DEV, gen)                                     # K no multiple of 16, rows side by side
    v = torch.randint(0, 120, (rows, 50), generator=gen, device=DEV).to(torch.uint8).view(E4M3)
    quantized.linear8(v, s, odd, out)
    check_product(out, v.double() * s.double()[:, None], dense8(odd), None)


@pytest.mark.parametrize("rows", [1, 8, 40, 300])
def test_what_lies_behind_a_row_is_not_read(rows):
    """NaN in the padding of rows and weights, and in rows behind the last."""
    gen = _gen(rows)
    for k in (5, 100, 130):
        w, (q, s) = random_weights8(33, k, DEV, gen), random_rows8(rows, k, DEV, gen)
        pitch = q.stride(0)
        wide = torch.full((rows + 3, pitch), 127, dtype=torch.uint8, device=DEV)
        wide[:rows, :k] = q.view(torch.uint8)
        values = torch.full((40, pitch), 127, dtype=torch.uint8, device=DEV)
        values[:33, :k] = w.values.view(torch.uint8)
        padded = quantized.Weights8(values.view(E4M3)[:33, :k], w.scales)
        out = torch.empty(rows, 33, device=DEV)
        quantized.linear8(wide.view(E4M3)[:rows, :k], s, padded, out)
        check_product(out, q.double() * s.double()[:, None], dense8(w), None)


@pytest.mark.parametrize("rows", [2, 8, 40, 300])
def test_infinities_and_nan_stay_in_their_rows(rows):
    gen = _gen(rows)
    nan, inf = float("nan"), float("inf")
    w4, w8 = random_weights4(50, 256, 64, DEV, gen), random_weights8(50, 256, DEV, gen)
    w4 = quantized.Weights4(w4.codes & ~0x00080008 | 0x00070007, torch.ones(50, 4, device=DEV).to(E4M3), w4.scales)
    for dtype in (torch.float32, torch.bfloat16):
        a = _randn(gen, rows, 256).to(dtype)
        clean = torch.empty(rows, 50, device=DEV)
        quantized.linear4(a, w4, clean)
        out = torch.empty_like(clean)
        a[0, 17], a[1, 255] = nan, inf
        quantized.linear4(a, w4, out)
        assert torch.isnan(out[0]).all() and not torch.isfinite(out[1]).any()
        assert torch.equal(out[2:], clean[2:])
        a[1, 255] = 1e30                                      # large, but a number
        a[0] = 0.0
        quantized.linear4(a, w4, out)
        check_product(out[1:], a[1:].double(), dense4(w4), None, 3)
        assert (out[0] == 0).all()
    q, s = random_rows8(rows, 256, DEV, gen)
    clean = torch.empty(rows, 50, device=DEV)
    quantized.linear8(q, s, w8, clean)
    out = torch.empty_like(clean)
    q.view(torch.uint8)[0, 100] = 127
    s[1] = inf
    quantized.linear8(q, s, w8, out)
    assert torch.isnan(out[0]).all() and not torch.isfinite(out[1]).any() and torch.equal(out[2:], clean[2:])


def test_a_row_does_not_depend_on_the_others():
    """The same row alone among zeros and among others, in steps that one kernel takes."""
    gen = _gen()
    w4, w8 = random_weights4(300, 512, 64, DEV, gen), random_weights8(300, 512, DEV, gen)
    for rows in (3, 40, 300):
        a = _randn(gen, rows, 512).bfloat16()
        q, s = random_rows8(rows, 512, DEV, gen)
        y4, y8 = torch.empty(rows, 300, device=DEV), torch.empty(rows, 300, device=DEV)
        quantized.linear4(a, w4, y4)
        quantized.linear8(q, s, w8, y8)
        a2, q2 = torch.zeros_like(a), torch.zeros_like(q.view(torch.uint8)).view(E4M3)
        a2[1], q2.view(torch.uint8)[1] = a[1], q.view(torch.uint8)[1]
        z4, z8 = torch.empty_like(y4), torch.empty_like(y8)
        quantized.linear4(a2, w4, z4)
        quantized.linear8(q2, s, w8, z8)
        assert torch.equal(y4[1], z4[1]) and torch.equal(y8[1], z8[1])


def test_packing_is_the_same_on_every_device():
    gen = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        w = (torch.randn(300, 1024, generator=gen) * 0.05).to(dtype)
        for group in (32, 128):
            here, there = quantized.Weights4.pack(w, group), quantized.Weights4.pack(w.to(DEV), group)
            assert torch.equal(here.codes, there.codes.cpu()) and torch.equal(here.scales, there.scales.cpu())
            assert torch.equal(here.group_scales.view(torch.uint8), there.group_scales.view(torch.uint8).cpu())
        here, there = quantized.Weights8.pack(w), quantized.Weights8.pack(w.to(DEV))
        assert torch.equal(here.values.view(torch.uint8), there.values.view(torch.uint8).cpu())
        assert torch.equal(here.scales, there.scales.cpu())


def _layer8(x, delta, gain, up, down, bufs):
    quantized.add_rmsnorm8(x, delta, gain, 1e-5, bufs["q"], bufs["s"])
    quantized.linear8(bufs["q"], bufs["s"], up, bufs["both"])
    quantized.glu8(bufs["both"], bufs["h"], bufs["hs"])
    quantized.linear8(bufs["h"], bufs["hs"], down, x, add=x)


def _layer_parts(rows, width, inter, seed):
    gen = _gen(seed)
    up = quantized.Weights8.pack(_randn(gen, 2 * inter, width) * width ** -0.5)
    down = quantized.Weights8.pack(_randn(gen, width, inter) * inter ** -0.5)
    x, delta = _randn(gen, rows, width), _randn(gen, rows, width).bfloat16()
    gain = 1 + 0.1 * _randn(gen, width)
    bufs = {"q": quantized.new_rows8(rows, width, DEV), "s": torch.empty(rows, device=DEV),
            "both": torch.empty(rows, 2 * inter, dtype=torch.bfloat16, device=DEV),
            "h": quantized.new_rows8(rows, inter, DEV), "hs": torch.empty(rows, device=DEV)}
    return x, delta, gain, up, down, bufs


@pytest.mark.parametrize("rows", [1, 8, 50, 333])
@pytest.mark.parametrize("width,inter", [(768, 2048), (100, 270)])
def test_a_feed_forward_in_8_bits(rows, width, inter):
    """Norm, product, gated pair, product into the residual: each stage against the 64-bit form of what the
    stage before it left."""
    x, delta, gain, up, down, b = _layer_parts(rows, width, inter, rows)
    before = x.clone()
    _layer8(x, delta, gain, up, down, b)
    total, y = exact_norm(before, delta, gain, 1e-5)
    check_rows8(b["q"], b["s"], y, "norm")
    check_product(b["both"], b["q"].double() * b["s"].double()[:, None], dense8(up), None, what="up")
    check_rows8(b["h"], b["hs"], exact_glu(b["both"], None), "pair")
    # (the residual was rounded once before it was added to)
    check_product(x, b["h"].double() * b["hs"].double()[:, None], dense8(down), before + delta.float(), what="down")


@pytest.mark.parametrize("rows", [1, 8, 50, 333])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_feed_forward_over_4_bits(rows, dtype):
    """The framework's own norm and gated pair around two products over 4-bit weights."""
    from crucible_b200 import ops
    gen = _gen(rows)
    width, inter, t = 768, 2048, DTYPES[dtype]
    up = quantized.Weights4.pack(_randn(gen, 2 * inter, width) * width ** -0.5, 64)
    down = quantized.Weights4.pack(_randn(gen, width, inter) * inter ** -0.5, 32)
    x, gain = _randn(gen, rows, width), 1 + 0.1 * _randn(gen, width)
    h, both, act = (torch.empty(rows, n, dtype=t, device=DEV) for n in (width, 2 * inter, inter))
    before = x.clone()
    ops.rmsnorm(x, gain, 1e-5, h)
    quantized.linear4(h, up, both)
    ops.swiglu(both, act)
    quantized.linear4(act, down, x, add=x)
    passes = 3 if dtype == "f32" else 1
    check_product(both, h.double(), dense4(up), None, passes, "up")
    check_product(x, act.double(), dense4(down), before, passes, "down")


def test_captured_on_two_streams_and_replayed_at_once():
    """Graphs of the whole feed-forward, captured on streams of their own and replayed side by side: nothing that
    one call uses is another's."""
    sides = []
    for i, rows in enumerate((4, 4, 40, 40, 260)):
        x, delta, gain, up, down, b = _layer_parts(rows, 768, 2048, 5 + i)
        start = x.clone()
        _layer8(x, delta, gain, up, down, b)                      # eagerly: what the replays must give
        want = x.clone()
        x.copy_(start)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x.copy_(start)
            _layer8(x, delta, gain, up, down, b)
        sides.append((stream, graph, x, want, (start, delta, gain, up, down, b)))
    for _ in range(20):
        for stream, graph, *_rest in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _stream, _graph, x, want, _kept in sides:
        assert torch.equal(x, want)


def test_on_a_stream_that_is_not_the_default():
    gen = _gen()
    w = random_weights4(1000, 2048, 64, DEV, gen)
    a = _randn(gen, 20, 2048).bfloat16()
    out = torch.empty(20, 1000, device=DEV)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            a.mul_(2)                                             # (the product reads what this wrote)
            quantized.linear4(a, w, out)
    stream.synchronize()
    check_product(out, a.double(), dense4(w), None)


def test_long_sums_keep_32_bits():
    """A sum of 16,384 like products, far beyond what an accumulator of fewer bits would hold."""
    k = 16384
    for rows in (1, 40, 300):
        q, s = torch.ones(rows, k, device=DEV).to(E4M3), torch.ones(rows, device=DEV)
        w8 = quantized.Weights8(torch.ones(130, k, device=DEV).to(E4M3), torch.ones(130, device=DEV))
        q.view(torch.uint8)[:, 1::2] = 0x10                       # 2^-5 beside 1: lost if few bits are kept
        out = torch.empty(rows, 130, device=DEV)
        quantized.linear8(q, s, w8, out)
        assert (out == k / 2 * (1 + 2.0 ** -5)).all()
        w4 = quantized.Weights4(torch.full((130, k // 8), -0x66666667, dtype=torch.int32, device=DEV),    # codes 9: one
                                torch.ones(130, k // 32, device=DEV).to(E4M3), torch.ones(130, device=DEV))
        a = q.float()
        for dtype in (torch.float32, torch.bfloat16):
            quantized.linear4(a.to(dtype), w4, out)
            assert (out == k / 2 * (1 + 2.0 ** -5)).all()


def test_the_largest_and_small_32_bit_rows_are_exact():
    """One weight of one: the row's number comes out as it went in, all 24 bits of it."""
    for rows in (1, 20, 300):
        codes = torch.full((20, 8), -0x77777778, dtype=torch.int32, device=DEV)                 # codes 8: zero
        codes[:, 3] = -0x77777777                                                              # k = 24: code 9
        w = quantized.Weights4(codes, torch.ones(20, 2, device=DEV).to(E4M3), torch.ones(20, device=DEV))
        a = _randn(_gen(), rows, 64)
        a[0, 24], a[-1, 24] = torch.finfo(torch.float32).max, 1.2345678e-30
        out = torch.empty(rows, 20, device=DEV)
        quantized.linear4(a, w, out)
        assert torch.equal(out, a[:, 24:25].expand(rows, 20))


@pytest.mark.parametrize("rows", [1, 20, 50, 100, 300])
@pytest.mark.parametrize("form", [None, "tiles", "pairs"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_float32_results_of_a_long_k_are_not_cut_off(rows, form, dtype, monkeypatch):
    """The tensor cores cut sums towards zero at every addition: with one sum over K = 16,384 the result was off by
    5e-6 of its norm.  In sums of 2,048 at most, 128 additions of at most 2^-23 of the sum each, half that on the
    average and the sum two thirds of its last value: 5e-6 / 8; float32 additions of 8 of them add 2^-24 each."""
    monkeypatch.setattr(quantized, "FORM", form)
    gen = _gen(rows)
    k = 16384
    w = quantized.Weights4.pack(_randn(gen, 260, k) * 0.02, 64)
    a = _randn(gen, rows, k).to(DTYPES[dtype])
    out = torch.empty(rows, 260, device=DEV)
    quantized.linear4(a, w, out)
    want = a.double() @ dense4(w).t()
    assert float((out.double() - want).norm() / want.norm()) <= 1e-6
    check_product(out, a.double(), dense4(w), None, 3 if dtype == "f32" else 1)


def test_every_form_on_streams_of_its_own():
    """Products of all forms side by side, eagerly, again and again: each gives what it gives alone."""
    gen = _gen()
    jobs = []
    for rows, n, k, dtype in ((1, 3000, 1024, "bf16"), (8, 9500, 512, "bf16"), (40, 2000, 2048, "bf16"), (300, 5000, 768, "bf16"),
                              (3, 900, 640, "f32"), (50, 1500, 4096, "f32"), (700, 1280, 512, "bf16")):
        w = random_weights4(n, k, 64, DEV, gen)
        a = _randn(gen, rows, k).to(DTYPES[dtype])
        out = torch.empty(rows, n, device=DEV)
        jobs.append((lambda a=a, w=w, out=out: quantized.linear4(a, w, out), out))
    for rows, n, k in ((1, 700, 768), (20, 4000, 2048), (64, 2048, 4096), (500, 3000, 1024)):
        w, (q, s) = random_weights8(n, k, DEV, gen), random_rows8(rows, k, DEV, gen)
        out = torch.empty(rows, n, device=DEV)
        jobs.append((lambda q=q, s=s, w=w, out=out: quantized.linear8(q, s, w, out), out))
    for call, _out in jobs:
        call()
    want = [out.clone() for _call, out in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _, out in jobs:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (call, _out) in zip(streams, jobs):
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    for (_call, out), right in zip(jobs, want):
        assert torch.equal(out, right)


def test_no_kernel_gave_up():
    """Runs last here: no bounded wait of the kernels above ran out."""
    from crucible_b200.ops import tensor_core
    tensor_core.check_status(DEV)
