"""Portions over the cache in 4 bits, in either form: errors held against the results' own size, and every border of what a row
sees against a key that stands out."""
import pytest
import torch

import cache4_cases as cc
import cache4_exact as ce

pytestmark = pytest.mark.gpu


def _attend(case, q, scale, **more):
    from crucible_b200.ops import cache4
    out = torch.full((q.shape[0], case.heads * case.dim), 7.0, dtype=q.dtype, device=q.device)
    cache4.attention4(q, out, case.heads, scale, case.batch, case.pages, **more)
    return out


@pytest.mark.parametrize("laid_out", [True, False])
@pytest.mark.parametrize("dim,group,n_rep,kv_heads,page,requests,window", [
    (64, 64, 3, 2, 16, [(0, 70)], None), (64, 32, 4, 1, 16, [(5, 100), (0, 65)], None), (128, 64, 4, 2, 16, [(200, 40)], None),
    (128, 128, 4, 1, 24, [(3000, 70), (5, 90), (64, 66)], 130), (128, 32, 4, 1, 64, [(3000, 70)], None),
    (64, 64, 8, 1, 16, [(0, 1100)], None), (128, 64, 2, 4, 16, [(0, 700), (900, 300)], 500)])
def test_errors_as_a_whole(dim, group, n_rep, kv_heads, page, requests, window, laid_out, monkeypatch):
    """(With keys, values and p in bfloat16 inside these are 0.0033 and more, with a scale that is off by 2 % 0.03.)"""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
    case = cc.Case(requests, dim=dim, group=group, n_rep=n_rep, kv_heads=kv_heads, page=page, seed=dim + n_rep + page)
    q = case.queries()
    ce.assert_as_a_whole(_attend(case, q, dim ** -0.5, window=window), ce.attention(case, q, dim ** -0.5, window), case.heads)


@pytest.mark.parametrize("laid_out", [True, False])
@pytest.mark.parametrize("dim,page,window,requests", [
    (64, 16, None, [(0, 140), (100, 70)]), (128, 16, None, [(60, 70), (127, 66)]), (64, 24, 70, [(90, 140), (0, 80)]),
    (128, 64, 64, [(200, 130), (63, 65)]), (64, 16, 65, [(64, 64), (191, 70)])])
def test_a_key_that_stands_out_at_every_border(dim, page, window, requests, laid_out, monkeypatch):
    """Equal scores, and one key whose values are a hundred times the others': each row sees it or does not, whole."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
    for r, (held, new) in enumerate(requests):
        last = held + new - 1
        places = {0, held - 1, held, held + 1, held + new // 2, last - 1, last, 63, 64, 127, 128, 191, 192}
        if window is not None:
            places |= {held - window, held - window + 1, last - window, last - window + 1}
        for place in sorted(p for p in places if 0 <= p <= last):
            case = cc.Case(requests, dim=dim, group=64, n_rep=2, kv_heads=2, page=page, seed=85 + place)
            at = int(case.table[r, place // page])
            case.pages.scales[1, at, :, place % page] *= 100
            q = torch.zeros(case.rows, case.heads * dim, dtype=torch.bfloat16, device=case.device)
            got, want = _attend(case, q, dim ** -0.5, window=window), ce.attention(case, q, dim ** -0.5, window)
            # (a result's rounding, 2^-8 of it at most, and p and v at eleven bits)
            error, size = (((t ** 2).view(case.rows, case.heads, dim).mean(dim=2)).sqrt() for t in (got.double() - want, want))
            assert bool((error <= (2.0 ** -8 + 2.0 ** -10) * size).all()), (r, place, float((error / size).max()))


@pytest.mark.parametrize("larger", [2.0 ** 10, 2.0 ** 24])
def test_vast_numbers_at_a_later_position_are_not_noticed_before_it(larger, monkeypatch):
    """Keys and values go into float16 by a power of two that follows the largest: exactly, within the range that is said."""
    from crucible_b200.ops import cache4
    for laid_out in (True, False):
        monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
        case = cc.Case([(30, 90), (0, 70)], dim=64, group=32, n_rep=4, kv_heads=2, seed=87)
        q = case.queries()
        before = _attend(case, q, 0.125)
        for place, first in ((100, 70), (119, 89), (75, 45)):           # (the row from which on it is seen)
            kept = case.pages.scales.clone()
            case.pages.scales[:, int(case.table[0, place // 16]), :, place % 16] *= larger
            got = _attend(case, q, 0.125)
            case.pages.scales.copy_(kept)
            assert torch.equal(got[:first], before[:first]) and torch.equal(got[90:], before[90:])
            assert torch.isfinite(got).all() and not torch.equal(got[first:90], before[first:90])
