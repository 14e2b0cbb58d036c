"""The cache in 4 bits, host side: what a batch and its operators refuse or hold to."""
import pytest
import torch


def _batch(rows, new, held):
    from crucible_b200.ops import cache4
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    return cache4.Batch(i(rows), i(rows), i(len(new) + 1), i(len(new)), i(len(new), 2), new, held)


def test_requests_of_more_tokens_than_there_are_rows():
    """Rows that no tensor has are refused here, not left to the kernels; rows behind the last request's are fine."""
    from crucible_b200.ops import KernelError
    for rows, new in ((3, [1, 100]), (3, [4]), (3, [1, 1, 1, 1]), (0, [1]), (5, [2, 2, 2])):
        with pytest.raises(KernelError, match="tokens, but it has"):
            _batch(rows, new, [0] * len(new))
    for rows, new in ((3, [1, 2]), (8, [1, 2]), (4, [4]), (3, [1, 1, 1])):
        assert _batch(rows, new, [7] * len(new)).rows == rows


def test_portions_of_prompts_are_told_from_decoded_tokens():
    """However few tokens a portion has left to it, and whatever stands before it in the step."""
    from crucible_b200.engine.scheduler import Request, Scheduler, SchedulerOptions
    from test_scheduler import FakeExecutor, greedy

    class Seen(FakeExecutor):
        def step(self, entries):
            seen.append([(e.request, len(e.tokens), e.prompt, e.decoded) for e in entries])
            return super().step(entries)
    seen = []
    s = Scheduler(Seen(n_pages=64), SchedulerOptions(max_batch=4, prefill_token_budget=11))
    s.submit(Request("a", list(range(10)), greedy(4)))
    s.submit(Request("b", list(range(3)), greedy(4)))
    s.submit(Request("c", [5], greedy(2)))
    s.run_to_completion()
    assert seen[0] == [("a", 10, True, False), ("b", 1, True, False)]
    assert seen[1] == [("a", 1, False, True), ("c", 1, True, False), ("b", 2, True, False)]
    assert all(decoded == (not prompt) for step in seen for _, _, prompt, decoded in step)
    assert sum(n for step in seen for _, n, prompt, _ in step if prompt) == 14
    assert sum(decoded for step in seen for *_, decoded in step) == 3 + 3 + 1


def test_steps_of_unlike_picks_are_captured_apart():
    from crucible_b200.engine.context import HostStep
    keys = {HostStep(list("ab"), [1, 1], [20, 9], [21, 10], [0, 1], picking).shape_key() for picking in (None, 0, 1, 2)}
    assert len(keys) == 4
    assert HostStep(list("ab"), [1, 1], [20, 9], [21, 10], [0, 1]).shape_key() in keys


def test_scales_that_float32_does_not_hold():
    """Nothing, or infinity, in float32: refused (and before anything is asked of a GPU)."""
    from crucible_b200.ops import KernelError, cache4
    pages = cache4.Pages4.new(2, 16, 1, 64, 32, device="cpu")
    q = torch.zeros(3, 64)
    for scale in (1e-50, 1e-46, 1e-39, 1e39, 1e300, 3e38):
        with pytest.raises(KernelError, match="scale"):
            cache4.attention4(q, q.clone(), 1, scale, _batch(3, [1, 2], [0, 4]), pages)
    for scale in (2e-38, 1e-20, 1.0, 1e37):
        with pytest.raises(KernelError, match="CUDA"):
            cache4.attention4(q, q.clone(), 1, scale, _batch(3, [1, 2], [0, 4]), pages)


def test_a_number_is_off_by_half_a_step_and_no_more():
    """Of the step as it is rounded: the largest number of a group, which its rounding may leave 15.06 steps above the low, is
    within the half, too.  (On top float32's rounding of x - low and of its product with the inverse: 16 steps of 3 * 2^-24.)"""
    import cache4_cases as cc
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(20000, 128, generator=gen).float().double() * torch.logspace(-6, 6, 20000)[:, None].float().double()
    x[::3] += 100 * torch.randn(len(x[::3]), 1, generator=gen).float().double() * x[::3].abs().amax(dim=1, keepdim=True)
    x = x.float().double()
    for group in (32, 64, 128):
        code, step, low = cc.coded(x, group)
        step = step.double().repeat_interleave(group, 1)
        got = code.double() * step + low.double().repeat_interleave(group, 1)
        assert bool(((got - x).abs() <= step * (0.5 + 1e-5)).all()), float(((got - x).abs() / step).max())
