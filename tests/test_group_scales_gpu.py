"""Each group's scale by itself: rows that are zero but in one group, so that no other group's products hide a wrong one."""
import pytest
import torch

from crucible_b200.ops import quantized
from quantized_cases import check_product, dense4, random_weights4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("form,rows,dtype", [("few", 8, "bf16"), ("few", 16, "f32"), ("ring", 1, "bf16"), ("ring", 8, "bf16"),
                                             ("ring", 16, "bf16"), ("ring", 5, "f32"), ("tiles", 32, "bf16"), ("tiles", 64, "bf16"),
                                             ("tiles", 250, "bf16"), ("tiles", 20, "f32"), ("tiles", 60, "f32"),
                                             ("pairs", 32, "bf16"), ("pairs", 250, "bf16")])
@pytest.mark.parametrize("k,group", [(256, 32), (1280, 160), (2080, 32), (2304, 96), (4096, 64), (4096, 128), (8448, 256), (8192, 4096)])
def test_a_group_alone(form, rows, dtype, k, group, monkeypatch):
    monkeypatch.setattr(quantized, "FORM", form)
    gen = torch.Generator(device=DEV).manual_seed(k + group)
    w = random_weights4(150, k, group, DEV, gen)
    weights = dense4(w)
    passes = 3 if dtype == "f32" else 1
    for first in range(0, k // group, rows):
        a = torch.zeros(rows, k, device=DEV)
        for i in range(min(rows, k // group - first)):
            at = (first + i) * group
            a[i, at:at + group] = torch.randn(group, generator=gen, device=DEV)
        a = a.to(torch.float32 if dtype == "f32" else torch.bfloat16)
        out = torch.empty(rows, 150, device=DEV)
        quantized.linear4(a, w, out)
        # (as many additions as K has, but those of zeros lose nothing: the bound of a K of one group and the sums of the shares)
        want, size = a.double() @ weights.t(), a.double().abs() @ weights.abs().t()
        bound = (passes * -(-group // 16) + 32) * 2.0 ** -23 * size
        assert ((out.double() - want).abs() <= bound + want.abs() * 2.0 ** -24).all(), f"groups from {first}"
        check_product(out, a.double(), weights, None, passes)


def test_no_kernel_gave_up():
    from crucible_b200.ops import tensor_core
    tensor_core.check_status(DEV)
