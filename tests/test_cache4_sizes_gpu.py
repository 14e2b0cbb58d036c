"""Attention over the cache in 4 bits: numbers at the ends of what the types hold, and arguments at the ends of theirs."""
import pytest
import torch

import cache4_cases as cc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _attend(case, q, scale, **more):
    from crucible_b200.ops import cache4
    out = torch.full((q.shape[0], case.heads * case.dim), 7.0, dtype=q.dtype, device=q.device)
    cache4.attention4(q, out, case.heads, scale, case.batch, case.pages, **more)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1.0, 1e3, 1e9, 1e20, 1e30])
def test_values_without_a_step(size, dtype):
    """Groups whose numbers are all alike (a step of zero), whatever their size; among them one that is not."""
    for held, uneven in ((0, False), (700, False), (700, True)):
        case = cc.Case([(held, 1), (held // 2, 2)], dim=64, group=32, dtype=dtype, seed=61)
        scales = case.pages.scales[1]
        scales[..., 0] = 0
        scales[..., 1] = (size * case.normal(*scales.shape[:-1])).to(BF16)
        if uneven:
            scales[int(case.table[0, 30]), :, 5, 1, 0] = 0.25
        q = case.queries()
        want, most = case.attention(q, 0.125)
        cc.assert_attention(_attend(case, q, 0.125), want, most, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", [1.0, 1e6, 1e12, 1e20, 1e30])
def test_values_of_nothing_beside_vast_ones(size, dtype, monkeypatch):
    """Keys whose values are all zero count in the weights, before, between and behind others, in one block or in many."""
    from crucible_b200.ops import cache4
    deal = cache4._shares
    for held, zeros in ((40, (0, 32)), (40, (8, 41)), (300, (0, 128)), (300, (100, 301)), (3000, (0, 1500)), (3000, (1000, 2500))):
        for dealt in (deal, lambda *a: (1, 0, 1.0), lambda *a: (2, 0, 1.0), lambda *a: (1, 8, 1.0)):
            monkeypatch.setattr(cache4, "_shares", dealt)
            case = cc.Case([(held, 1)], dim=64, group=32, dtype=dtype, seed=67)
            case.pages.scales[1] *= size
            for j in range(*zeros):
                case.pages.scales[1, int(case.table[0, j // 16]), :, j % 16] = 0
            q = case.queries(0.3)
            want, most = case.attention(q, 0.125)
            cc.assert_attention(_attend(case, q, 0.125), want, most, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("stretch,scale", [(1e-30, 1e-16), (1e-36, 1e-5), (1e-30, 1e-37), (1.0, 1e-37)])
def test_scores_of_next_to_nothing(stretch, scale, dtype):
    """Queries times the scale under float32's least number: all keys count alike, masked ones not at all."""
    case = cc.Case([(200, 1), (90, 2)], dim=64, group=32, dtype=dtype, seed=63)
    q = case.queries(stretch)
    want, most = case.attention(q, scale)
    cc.assert_attention(_attend(case, q, scale), want, most, dtype)
    want, most = case.attention(q, scale, window=37)
    cc.assert_attention(_attend(case, q, scale, window=37), want, most, dtype)


@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 62])
def test_windows_beyond_every_context(window, monkeypatch):
    from crucible_b200.ops import cache4
    for laid_out in (False, True):
        monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
        case = cc.Case([(100, 40), (0, 30)], dim=64, group=64, n_rep=4, kv_heads=1, seed=65)
        q = case.queries()
        assert torch.equal(_attend(case, q, 0.125, window=window), _attend(case, q, 0.125))
