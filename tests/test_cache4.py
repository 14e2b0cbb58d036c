"""The cache in 4 bits, host side: its format, what its operators refuse, and how keys are dealt to blocks."""
import pytest
import torch

import cache4_cases as cc

BF16, F32 = torch.bfloat16, torch.float32


def _ops():
    from crucible_b200.ops import KernelError, cache4
    return cache4, KernelError


def _pages(dim=64, group=32, page=16, kv=2, bounds=False, n=3):
    cache4, _ = _ops()
    return cache4.Pages4.new(n, page, kv, dim, group, bounds=bounds, device="cpu")


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _batch(new=(1, 2), held=(4, 0), pages=2):
    cache4, _ = _ops()
    rows = sum(new)
    return cache4.Batch(torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32),
                        torch.zeros(len(new) + 1, dtype=torch.int32), torch.zeros(len(new), dtype=torch.int32),
                        torch.zeros(len(new), pages, dtype=torch.int32), list(new), list(held))


def test_rows_lie_in_memory_as_the_format_says():
    """Every feature has bits of its own, and what is packed comes out again."""
    for dim in (64, 128, 192, 256):
        codes = torch.randint(0, 16, (5, dim))
        assert torch.equal(cc.unpacked(cc.packed(codes)), codes)
        one = torch.zeros(dim, dim, dtype=torch.int64)
        one.fill_diagonal_(15)
        lit = cc.packed(one)
        assert ((lit == 15) | (lit == 240) | (lit == 0)).all() and (lit.sum(dim=0) == 255).all()
    word = cc.packed(torch.arange(64)[None] // 8)[0, :4].tolist()        # the first word: features 0, 8, .., 56
    assert word == [0x10, 0x54, 0x32, 0x76]


def test_a_number_is_off_by_half_a_step():
    x = torch.randn(400, 128).float().double() * torch.logspace(-6, 6, 400)[:, None].float().double()
    for group in (32, 64, 128):
        code, step, low = cc.coded(x, group)
        got = code.double() * step.double().repeat_interleave(group, 1) + low.double().repeat_interleave(group, 1)
        assert ((got - x).abs() <= step.double().repeat_interleave(group, 1) * (0.5 + 15 * 2.0 ** -8 + 1e-5)).all()


def test_pools_that_are_refused():
    cache4, KernelError = _ops()
    good = _pages()
    assert (good.n_pages, good.kv_heads, good.page_tokens, good.head_dim, good.group) == (3, 2, 16, 64, 32)
    codes, scales = good.codes, good.scales
    for bad in (codes.to(torch.int32), codes[0], codes.transpose(1, 2), codes[..., :24], codes[:1]):
        with pytest.raises(KernelError, match="codes"):
            cache4.Pages4(bad, scales)
    for bad in (scales.float(), scales[..., :1, :], scales[:, :2], scales[..., 0], scales.transpose(2, 3)):
        if tuple(bad.shape) == (2, 3, 2, 16, 1, 2):
            cache4.Pages4(codes, bad.contiguous())                       # one group of 64: as good
            bad = bad.transpose(1, 2)
        with pytest.raises(KernelError, match="scales"):
            cache4.Pages4(codes, bad)
    kept = _pages(bounds=True)
    for b, s in ((kept.bounds, None), (None, kept.bound_scales), (kept.bounds.float(), kept.bound_scales),
                 (kept.bounds[:2], kept.bound_scales), (kept.bounds, kept.bound_scales.double())):
        with pytest.raises(KernelError, match="bounds"):
            cache4.Pages4(codes, scales, b, s)
    for args in ((0, 16, 2, 64), (3, 0, 2, 64), (3, 16, 0, 64), (3, 16, 2, 80), (3, 16, 2, 512), (3, 16, 2, 64, 128),
                 (3, 16, 2, 64, 16), (3, 16, 2, 192, 128)):
        with pytest.raises(KernelError):
            cache4.Pages4.new(*args, device="cpu")
    whole = torch.zeros(codes.numel() + 8, dtype=torch.uint8)
    with pytest.raises(KernelError, match="16 bytes"):
        cache4.Pages4(whole[8:].view(codes.shape), scales)
    with pytest.raises(KernelError):
        good.values(torch.float16)
    with pytest.raises(KernelError, match="CUDA"):
        good.values()
    with pytest.raises(KernelError, match="no bounds"):
        good.bound_values()


def test_batches_that_are_refused():
    cache4, KernelError = _ops()
    ok = _batch((1, 1, 5), (3, 0, 7))
    assert (ok.most_new, ok.reach, ok.lead, ok.requests) == (5, 12, 2, 3)
    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    good = dict(positions=i(3), row_request=i(3), row_start=i(3), first_pos=i(2), table=i(4).view(2, 2), new_tokens=[1, 2],
                held_tokens=[0, 4])
    cache4.Batch(**good)
    for name, bad in (("positions", i(4)), ("positions", i(3).long()), ("row_request", i(3).float()), ("row_start", i(2)),
                      ("first_pos", i(3)), ("table", i(4)), ("table", i(6).view(3, 2)), ("table", i(4).view(2, 2).t()),
                      ("table", i(0).view(2, 0)), ("positions", i(6)[::2]), ("new_tokens", [1, 0]), ("new_tokens", [3]),
                      ("held_tokens", [0]), ("held_tokens", [-1, 0]), ("new_tokens", [])):
        with pytest.raises(KernelError):
            cache4.Batch(**{**good, name: bad})


def test_calls_that_are_refused():
    cache4, KernelError = _ops()
    pages, batch = _pages(bounds=True), _batch()
    rows, heads = 3, 4
    q, out = torch.zeros(rows, heads * 64), torch.zeros(rows, heads * 64)
    qkv = torch.zeros(rows, (heads + 4) * 64)
    cos = torch.zeros(9, 32)
    picks = torch.zeros(rows, 2, 4, dtype=torch.int32)

    def attend(**kw):
        a = dict(q=q, out=out, n_heads=heads, scale=0.1, batch=batch, pages=pages, window=None, picks=None)
        a.update(kw)
        cache4.attention4(**a)

    def append(**kw):
        a = dict(qkv=qkv, q=q, n_heads=heads, cos=cos, sin=cos, batch=batch, pages=pages)
        a.update(kw)
        cache4.rope_append4(**a)

    def pick(**kw):
        a = dict(q=q, n_heads=heads, batch=batch, pages=pages, picks=picks)
        a.update(kw)
        cache4.pick_pages4(**a)

    for call in (attend, append, pick):                                  # all is well, but there is no GPU
        with pytest.raises(KernelError, match="CUDA device only"):
            call()
        with pytest.raises(KernelError):
            call(batch=_batch((1, 3)))
        with pytest.raises(KernelError):
            call(q=q[:, :-1])
        with pytest.raises(KernelError):
            call(q=q.double())
        with pytest.raises(KernelError):
            call(q=torch.zeros(heads * 64, rows).t())
        with pytest.raises(KernelError):
            call(q=torch.zeros(1, heads * 64).expand(rows, -1))
        with pytest.raises(KernelError):
            call(n_heads=0)
    for call in (attend, pick):
        with pytest.raises(KernelError, match="evenly"):
            call(n_heads=3, **({"q": q[:, :192], "out": out[:, :192]} if call is attend else {"q": q[:, :192]}))
        for bad in (picks.long(), picks[:0] if call is pick else picks[:2], picks[:, :1], picks[..., 0], picks.transpose(0, 1), picks[..., :0]):
            with pytest.raises(KernelError, match="picks"):
                call(picks=bad)
    for bad in (dict(out=out.bfloat16()), dict(out=out[:, :64]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(window=0), dict(window=-3), dict(picks=picks, window=8),
                dict(picks=picks, pages=_pages(page=24))):
        with pytest.raises(KernelError):
            attend(**bad)
    for bad in (dict(qkv=qkv[:, 1:]), dict(qkv=qkv.bfloat16()), dict(cos=None), dict(sin=cos[:8]), dict(cos=cos.double(), sin=cos.double()),
                dict(cos=torch.zeros(9, 33), sin=torch.zeros(9, 33)), dict(cos=cos.t(), sin=cos.t())):
        with pytest.raises(KernelError):
            append(**bad)
    for bad in (dict(pages=_pages()), dict(first=-1), dict(last=0), dict(first=2, last=3)):
        with pytest.raises(KernelError):
            pick(**bad)


def test_keys_are_dealt_to_as_many_blocks_as_there_is_room_for():
    cache4, _ = _ops()
    for resident in (296, 444, 592):
        for blocks in (1, 2, 8, 37, 148, 512, 700, 100000):
            for tiles in (1, 7, 8, 60, 500, 8192, 1 << 20):
                for total in (blocks * tiles, blocks + tiles):
                    shares, stream, us = cache4._shares(blocks, tiles, total, resident)
                    assert us > 2
                    assert shares in (1, 2, 4, 8) and (shares == 1 or stream == 0)
                    assert 0 <= stream <= resident and (stream == 0 or (blocks < 4 * resident and total >= 8))
                    assert shares == 1 or tiles > 4 * shares          # no block of a cluster without a round


def test_pages_are_scored_by_no_more_blocks_than_a_cluster_has():
    cache4, _ = _ops()
    assert cache4._pick_shares(1, 100000) == 8 and cache4._pick_shares(10000, 100000) == 1 and cache4._pick_shares(1, 200) == 1
