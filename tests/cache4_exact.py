"""Attention over the cache in 4 bits in 64 bits, whole requests at a time (long contexts), and how far results may be off as
a whole: the root of the mean square, which an error that all results share cannot pass under."""
from __future__ import annotations

import math

import torch


def attention(case, q, scale, window=None):
    """Results float64 [rows, heads * dim] of a `cache4_cases.Case` whose tables name a page for every key that is seen."""
    from cache4_cases import values
    rep, out, row = case.heads // case.kv_heads, torch.zeros(case.rows, case.heads, case.dim, dtype=torch.float64, device=case.device), 0
    for r, (held, new) in enumerate(case.requests):
        ids = case.table[r, :-(-(held + new) // case.page)].long()
        k, v = (values(case.pages.codes[i][ids], case.pages.scales[i][ids]).transpose(0, 1).flatten(1, 2) for i in (0, 1))
        key, place = torch.arange(k.shape[1], device=case.device), held + torch.arange(new, device=case.device)[:, None]
        hidden = key > place
        if window is not None:
            hidden = hidden | (key <= place - window)
        for h in range(case.heads):
            logits = q[row:row + new].double().view(new, case.heads, case.dim)[:, h] @ k[h // rep].t() * scale
            out[row:row + new, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1) @ v[h // rep]
        row += new
    return out.flatten(1)


# Rounding a result to bfloat16 is off by 2^-8 of itself at most, evenly spread: 2^-8 / sqrt(3) as a root of the mean square
# (if every result were just above a power of two; 0.0016 as a rule).  What is inside has eleven bits and more: p step, or p,
# v and k each by themselves, 2^-11 / sqrt(3) apiece and independent, so that they add as squares; scores of terms of up to
# 2^3 (in q, k of ordinary size) at eleven bits move p by 2^-8 / 4 and less.
ROUNDED = 2.0 ** -8 / math.sqrt(3.0)
INSIDE = math.sqrt(3 * (2.0 ** -11) ** 2 / 3 + (2.0 ** -10) ** 2)
AS_A_WHOLE = math.sqrt(ROUNDED ** 2 + INSIDE ** 2)


def assert_as_a_whole(got, want, heads, most=AS_A_WHOLE):
    """The root of the mean square error of every head, of that of its results."""
    error = ((got.double() - want) ** 2).view(want.shape[0], heads, -1).mean(dim=(0, 2)).sqrt()
    size = (want ** 2).view(want.shape[0], heads, -1).mean(dim=(0, 2)).sqrt()
    assert bool((error <= most * size).all()), f"{float((error / size).max())} of the results, at most {most}"
