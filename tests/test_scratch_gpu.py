"""What a call takes from torch's pool while it runs."""
import pytest
import torch

from crucible_b200.ops import quantized
from quantized_cases import check_product, dense4, random_weights4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows,n,k", [(24000, 64, 16384), (300, 40, 524288), (65537, 40, 2048)])
def test_float32_rows_over_4_bit_weights_take_512_mb_at_most(rows, n, k):
    gen = torch.Generator(device=DEV).manual_seed(rows)
    w = random_weights4(n, k, 64, DEV, gen)
    a = torch.randn(rows, k, generator=gen, device=DEV)
    out, plus = torch.empty(rows, n, device=DEV), torch.randn(rows, n, generator=gen, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    quantized.linear4(a, w, out, add=plus)
    assert torch.cuda.max_memory_allocated() - before <= 512 << 20
    weights = dense4(w)
    for at in (0, rows // 2 // 64 * 64 - 40, rows - 80):           # both ends, and where two parts may meet
        check_product(out[at:at + 80], a[at:at + 80].double(), weights, plus[at:at + 80], 3)
