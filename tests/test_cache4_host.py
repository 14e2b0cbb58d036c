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
