"""Captured steps over the cache in 4 bits, replayed with rows dealt to their requests in another way."""
import pytest
import torch

import cache4_cases as cc
import cache4_exact as ce

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _captured(case, window):
    from crucible_b200.ops import cache4
    q = case.queries()
    out = torch.empty_like(q)

    def step():
        cache4.attention4(q, out, case.heads, 0.125, case.batch, case.pages, window=window)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    return graph, q, out


def _dealt(case, requests):
    """The step's numbers on the device for these requests (held, new); the host's stay the capture's."""
    case.requests = requests
    starts = [0]
    for _, n in requests:
        starts.append(starts[-1] + n)
    case.rows = starts[-1]
    case.row_start.copy_(torch.tensor(starts))
    case.first_pos.copy_(torch.tensor([h for h, _ in requests]))
    case.positions[:case.rows] = torch.tensor([h + i for h, n in requests for i in range(n)], dtype=torch.int32, device=DEV)
    case.row_request.fill_(-1)
    case.row_request[:case.rows] = torch.tensor([r for r, (_, n) in enumerate(requests) for _ in range(n)], dtype=torch.int32,
                                                device=DEV)


def _check(case, graph, q, out, requests, window):
    _dealt(case, requests)
    out.fill_(7)
    graph.replay()
    want = ce.attention(case, q[:case.rows], 0.125, window)
    ce.assert_as_a_whole(out[:case.rows], want, case.heads)
    spread = []
    exact, most = case.attention(q[:case.rows], 0.125, window=window, spread=spread)
    cc.assert_attention_laid_out(out[:case.rows], exact, most, spread[0])
    assert (out[case.rows:] == 7).all()


def test_rows_that_move_between_requests_in_a_window(monkeypatch):
    """Other requests bring the most rows now, and reach more blocks of 64 tokens than theirs at the capture did."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    case = cc.Case([(700, 50), (640, 114)], dim=64, group=64, n_rep=2, kv_heads=1, page=16, seed=47)
    graph, q, out = _captured(case, 79)
    for requests in ([(461, 52), (560, 112)], [(600, 114), (640, 50)], [(63, 100), (1, 64)], [(636, 114), (703, 50)], [(0, 1), (0, 1)]):
        _check(case, graph, q, out, requests, 79)


@pytest.mark.parametrize("blocks", [3, 1])
def test_rows_that_move_between_requests_laid_out_one_at_a_time(blocks, monkeypatch):
    """Requests that are laid out, or (one alone has more blocks than that) walked, by themselves: one that brought few rows at the
    capture brings as many as the most now."""
    from crucible_b200.ops import cache4
    monkeypatch.setattr(cache4, "LAID_OUT", True)
    monkeypatch.setattr(cache4, "_MOST_BLOCKS", blocks * 64)
    case = cc.Case([(70, 40), (0, 110)], dim=64, group=64, n_rep=2, kv_heads=1, page=16, seed=49)
    graph, q, out = _captured(case, None)
    for requests in ([(0, 110), (70, 40)], [(5, 75), (20, 75)], [(30, 64), (0, 80)]):
        _check(case, graph, q, out, requests, None)
