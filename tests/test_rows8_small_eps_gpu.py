"""Norms in 8 bits whose eps is so small that a row of next to nothing has a large factor 1 / sqrt(mean + eps)."""
import pytest
import torch

from crucible_b200.ops import quantized
from quantized_cases import LEAST, TOP, check_rows8, exact_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("width", [5, 64, 768, 4096, 20000])
@pytest.mark.parametrize("eps", [1e-5, 1.4e-11, 1.5e-11, 1.6e-12, 1.8e-12, 1e-12, 1e-15, 1e-20])
def test_rows_of_next_to_nothing(width, eps):
    gen = torch.Generator(device=DEV).manual_seed(width)
    size = [0.0, 1e-36, 1e-33, 1e-30, 1e-25, 1e-20, 1e-10, 1.0]
    x = torch.randn(len(size), width, generator=gen, device=DEV) * torch.tensor(size, device=DEV)[:, None]
    x[1:, width // 2] = 0.0
    gain = 1 + 0.2 * torch.randn(width, generator=gen, device=DEV)
    q, s = quantized.new_rows8(len(size), width, DEV), torch.empty(len(size), device=DEV)
    quantized.add_rmsnorm8(x, None, gain, eps, q, s)
    # (eps as the kernel has it; squares below 2^-126 are nothing beside it)
    _total, y = exact_norm(x, None, gain, float(torch.tensor(eps, dtype=torch.float32)))
    assert (q[0].float() == 0).all() and float(s[0]) == pytest.approx(LEAST / TOP, rel=1e-6)
    assert (q[1:, width // 2].float() == 0).all()
    check_rows8(q, s, y, f"eps {eps}")
