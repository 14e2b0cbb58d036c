"""Attention over the cache in 4 bits where the numbers on the device are not those that the host was told of: both forms leave
alone what they have no rows for, and see the keys that there are."""
import pytest
import torch

import cache4_cases as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _attend(case, q, rows_behind, **more):
    """Results, and the rows behind the batch's of the tensors that they lie in."""
    from crucible_b200.ops import cache4
    whole = torch.full((case.batch.rows + rows_behind, case.heads * case.dim), 7.0, dtype=q.dtype, device=DEV)
    rows = torch.full_like(whole, float("nan"))
    rows[:case.batch.rows] = q
    cache4.attention4(rows[:case.batch.rows], whole[:case.batch.rows], case.heads, 0.125, case.batch, case.pages, **more)
    return whole[:case.batch.rows], whole[case.batch.rows:]


@pytest.mark.parametrize("laid_out", [True, False])
@pytest.mark.parametrize("window", [None, 50])
def test_rows_beyond_the_tensors(laid_out, window, monkeypatch):
    """Rows that begin before the first or end behind the last row of queries and results.  (All that could be reached by
    mistake is memory of these tensors' own.)"""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
    case = cc.Case([(30, 70), (64, 40), (100, 64)], dim=64, group=32, n_rep=4, kv_heads=2, seed=71)
    q, spread = case.queries(), []
    want, most = case.attention(q, 0.125, window=window, spread=spread)
    for starts, there in (([0, 70, 110, 174 + 60], 174), ([0, 70, 110, 1 << 30], 174), ([0, 70, 200, 230], 70),
                          ([-20, 70, 110, 174], (70, 174))):
        case.row_start.copy_(torch.tensor(starts))
        got, behind = _attend(case, q, 64, window=window)
        assert (behind == 7).all()
        first, last = there if isinstance(there, tuple) else (0, there)
        part = slice(first, last)
        check = cc.assert_attention_laid_out if laid_out else lambda *a: cc.assert_attention(*a[:3], torch.bfloat16)
        if starts[2] == 200:                     # (the second has 104 rows then, more than the most that the host was told of, 70:
            part = slice(0, 70)                  # which of these are worked on is not said)
        check(got[part], want[part], most[part], spread[0][part])
        assert (got[:first] == 7).all()


@pytest.mark.parametrize("laid_out", [True, False])
def test_positions_beyond_the_table(laid_out, monkeypatch):
    """Rows far behind all that the table has a place for see what there is, once."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", laid_out)
    case = cc.Case([(64, 64), (30, 70)], dim=64, group=64, n_rep=2, kv_heads=1, page=16, seed=73)      # eight pages, two blocks of 64
    for first in (64, 90, 128, 5000):
        case.first_pos.copy_(torch.tensor([first, 30]))
        case.positions[:64] = first + torch.arange(64, device=DEV)
        q, spread = case.queries(), []
        want, most = case.attention(q, 0.125, spread=spread)
        got, _ = _attend(case, q, 0)
        cc.assert_attention_laid_out(got, want, most, spread[0])
