"""Gated pairs of many long rows with and without a place to tell of waits that run out: two kernels, the same bits."""
import pytest
import torch

from crucible_b200.ops import build, quantized, tensor_core

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,rows,width", [("bf16", 295, 20000), ("bf16", 296, 20000), ("bf16", 600, 28800), ("bf16", 1024, 14336),
                                              ("f32", 296, 7176), ("f32", 1023, 14400), ("f32", 1100, 7168)])
@pytest.mark.parametrize("pair", [(None, 1.0, 0.0), (2.0, 1.25, 0.75)])
def test_the_same_bits(dtype, rows, width, pair, monkeypatch):
    gen = torch.Generator(device=DEV).manual_seed(rows + width)
    both = (2 * torch.randn(rows, 2 * width, generator=gen, device=DEV)).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    results = []
    for word in (tensor_core.status_word(torch.device(DEV)).data_ptr(), 0):
        monkeypatch.setattr(quantized, "_status", lambda dev: word)
        assert bool(build.load("rows8").cb_glu8_waits(dtype == "bf16", rows, width, word)) == (word != 0 and rows >= 296)
        q, s = quantized.new_rows8(rows, width, DEV), torch.full((rows,), -1.0, device=DEV)
        quantized.glu8(both, q, s, *pair)
        results.append((q.contiguous().view(torch.uint8), s))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    tensor_core.check_status(DEV)
