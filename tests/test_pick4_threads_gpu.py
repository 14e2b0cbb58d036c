"""Host threads that pick among pages of contexts of unlike lengths."""
import sys
import threading

import pytest
import torch

import cache4_cases as cc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_threads_pick_behind_short_and_long_contexts(monkeypatch):
    """The longer ones' scores take more shared memory than the others'; no launch is refused for another's sake.  (The entry
    point's calls are repeated by themselves: between the checks of whole ones two threads hardly ever meet.)"""
    from crucible_b200.ops import cache4
    cases = [cc.Case([(held, 1)], dim=64, group=64, n_rep=2, kv_heads=1, page=1, seed=81, bounds=True) for held in (100, 20000)]
    calls, at = [], cache4._at
    monkeypatch.setattr(cache4, "_at", lambda dev, call, *a: calls.append((call, a)) or at(dev, call, *a))
    kept = []
    for case in cases:
        case.pages.bounds.copy_(torch.randint(-127, 128, case.pages.bounds.shape, generator=case.gen, device=DEV, dtype=torch.int8))
        case.pages.bound_scales.fill_(0.01)
        q, picks = case.queries(), torch.empty(1, 1, 8, dtype=torch.int32, device=DEV)
        cache4.pick_pages4(q, case.heads, case.batch, case.pages, picks)
        kept.append((q, picks, picks.clone()))
    torch.cuda.synchronize()
    refused, start = [0] * 8, threading.Barrier(8)

    def run(i):
        stream = torch.cuda.Stream(DEV)
        call, args = calls[i % 2]
        start.wait()
        for n in range(10000):
            refused[i] += call(*args, stream.cuda_stream) != 0
            if n % 500 == 0:
                stream.synchronize()
        stream.synchronize()
    was = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
    finally:
        sys.setswitchinterval(was)
    assert refused == [0] * 8
    assert all(torch.equal(picks, want) for _, picks, want in kept)
