"""float32 results of long dot products over quantised weights.  The tensor cores cut off, towards zero, what an addition
leaves below the sum's last bit: a bfloat16 row by 4-bit weights of K = 16,384 in one sum came out 5e-6 of the result's norm
off, and that grows with the length of the sum.  Taken 2,048 of K at a time it is an eighth of that, 6.3e-7, whatever K is;
the additions of those sums, rounded, are 2^-24 each and of both signs: 1e-6 in all."""
import pytest
import torch

from crucible_b200.ops import quantized
from quantized_cases import E4M3, TOP, check_product, dense4, dense8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _check4(rows, n, k, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows + k)
    a = torch.randn(rows, k, generator=gen, device=DEV).to(DTYPES[dtype])
    w = quantized.Weights4.pack(torch.randn(n, k, generator=gen, device=DEV) * 0.02, 64)
    out = torch.empty(rows, n, device=DEV)
    quantized.linear4(a, w, out)
    few = min(n, 256)
    w = quantized.Weights4(w.codes[-few:], w.group_scales[-few:], w.scales[-few:])
    want = a.double() @ dense4(w).t()
    assert float((out[:, -few:].double() - want).norm() / want.norm()) <= 1e-6
    check_product(out[:, -few:], a.double(), dense4(w), None, 3 if dtype == "f32" else 1)


@pytest.mark.parametrize("rows,dtype", [(1, "bf16"), (8, "bf16"), (16, "bf16"), (1, "f32"), (5, "f32")])
def test_few_rows_by_many_features(rows, dtype):
    _check4(rows, 12032, 32768, dtype)


@pytest.mark.parametrize("block", [(1, 8), (1, 4), (2, 4), (2, 2)])
@pytest.mark.parametrize("shares", [1, 2])
@pytest.mark.parametrize("rows,dtype", [(1, "bf16"), (9, "bf16"), (2, "f32"), (3, "f32")])
def test_every_block_of_the_ring(block, shares, rows, dtype, monkeypatch):
    monkeypatch.setattr(quantized, "_rule", lambda *sizes: ("ring", *block, shares))
    _check4(rows, 100, 65536, dtype)
    _check4(rows, 100, 65536 + 1280, dtype)            # a last sum that is short


@pytest.mark.parametrize("k", [65536, 65536 + 2080 + 32])
@pytest.mark.parametrize("rows,dtype", [(1, "bf16"), (9, "bf16"), (2, "f32"), (9, "f32")])
def test_from_registers(k, rows, dtype, monkeypatch):
    monkeypatch.setattr(quantized, "FORM", "few")
    gen = torch.Generator(device=DEV).manual_seed(k)
    a = torch.randn(rows, k, generator=gen, device=DEV).to(DTYPES[dtype])
    w = quantized.Weights4.pack(torch.randn(40, k, generator=gen, device=DEV) * 0.02, 32)
    out = torch.empty(rows, 40, device=DEV)
    quantized.linear4(a, w, out)
    want = a.double() @ dense4(w).t()
    assert float((out.double() - want).norm() / want.norm()) <= 1e-6
    check_product(out, a.double(), dense4(w), None, 3 if dtype == "f32" else 1)


@pytest.mark.parametrize("rows", [1, 20, 33, 100])
@pytest.mark.parametrize("n,k", [(200, 262144), (20000, 24576), (20000, 32768), (600, 73728)])
def test_8_bit_rows(rows, n, k):
    """e4m3 products have 8 bits, and sums of them of 12,288 of K stay below the bound."""
    gen = torch.Generator(device=DEV).manual_seed(rows + k)
    x = torch.randn(rows, k, generator=gen, device=DEV)
    s = x.abs().amax(dim=1) / TOP
    q = (x / s[:, None]).clamp(-TOP, TOP).to(E4M3)
    w = quantized.Weights8.pack(torch.randn(n, k, generator=gen, device=DEV) * 0.02)
    out = torch.empty(rows, n, device=DEV)
    quantized.linear8(q, s, w, out)
    w = quantized.Weights8(w.values[-200:], w.scales[-200:])
    exact = q.double() * s.double()[:, None]
    want = exact @ dense8(w).t()
    assert float((out[:, -200:].double() - want).norm() / want.norm()) <= 1e-6
    check_product(out[:, -200:], exact, dense8(w), None)


def test_no_kernel_gave_up():
    from crucible_b200.ops import tensor_core
    tensor_core.check_status(DEV)
