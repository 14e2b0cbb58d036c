"""Attention over the cache in 4 bits: bfloat16 results that average very many keys, held against their own size."""
import pytest
import torch

import cache4_cases as cc
import cache4_exact as ce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("one_block", [False, True])
@pytest.mark.parametrize("size", [0.0, 1.0])
@pytest.mark.parametrize("dim,group,n_rep,requests", [
    (64, 64, 4, [(32000 + 37 * i, 1) for i in range(16)]), (128, 64, 8, [(131000, 1)]), (128, 128, 4, [(40000, 1), (70001, 3)]),
    (192, 32, 2, [(50000, 1)]), (256, 64, 4, [(33000, 2)])])
def test_means_of_many_keys(dim, group, n_rep, requests, size, one_block, monkeypatch):
    """Queries of zeros: a result is the mean of the values, 1 / sqrt(n) of one of them; a block that takes all keys by itself,
    and as many as the sizes ask for."""
    from crucible_b200.ops import cache4
    if one_block:
        monkeypatch.setattr(cache4, "_shares", lambda *a: (1, 0, 1.0))
    monkeypatch.setattr(cache4, "LAID_OUT", False)
    case = cc.Case(requests, dim=dim, group=group, n_rep=n_rep, kv_heads=1, page=16, seed=dim + n_rep)
    q = case.queries(size)
    out = torch.empty_like(q)
    cache4.attention4(q, out, case.heads, dim ** -0.5, case.batch, case.pages)
    ce.assert_as_a_whole(out, ce.attention(case, q, dim ** -0.5), case.heads)
