"""The cache in 4 bits on a device that is not the current one, after the same calls on the first."""
import pytest
import torch

import cache4_cases as cc

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(torch.cuda.device_count() < 2, reason="takes two devices")]


@pytest.mark.parametrize("laid_out", [True, False])
def test_portions_on_a_second_device(laid_out, monkeypatch):
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
    for device in ("cuda:0", "cuda:1"):
        for dim in (64, 128):
            case = cc.Case([(5, 1), (100, 70)], dim=dim, group=64, n_rep=2, kv_heads=1, seed=83, device=device, bounds=True)
            q, spread = case.queries(), []
            want, most = case.attention(q, 0.1, spread=spread)
            out = torch.empty_like(q)
            cache4.attention4(q, out, case.heads, 0.1, case.batch, case.pages)
            cc.assert_attention_laid_out(out, want, most, spread[0])
            picks = torch.empty(1, 1, 3, dtype=torch.int32, device=device)
            cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks)
            torch.cuda.synchronize(device)
