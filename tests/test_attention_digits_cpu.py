"""The bounds of _attention_digits notice what they are for: a forward pass in fp32 with P rounded to bf16 is inside them with a second
product for what the rounding left, and outside without it or with the remainder of the wrong columns."""
import math

import pytest
import torch

from _attention_bounds import visible
from _attention_digits import check_digits, output64

BF = torch.bfloat16


def _forward(q, k, v, mask, remainder):
    q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
    s = (q @ k.transpose(2, 3) / math.sqrt(q.shape[-1])).masked_fill(~mask, -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    hi = p.to(BF).float()
    lo = (p - hi).to(BF).float() if remainder != "none" else torch.zeros_like(p)
    if remainder == "wrong":
        lo = lo.roll(1, -1)
    return ((hi @ v + lo @ v) / p.sum(-1, keepdim=True)).transpose(1, 2).to(BF)


@pytest.mark.parametrize("T,window,sinks", [(300, 100, 0), (300, 2, 0), (517, 300, 4), (150, 150, 0)])
def test_the_second_product_counts(T, window, sinks):
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn(2, T, 4, 64, generator=g) for _ in range(3))
    q, k, v = (2 * q).to(BF), k.to(BF), v.to(BF)
    mask = visible(T, window, sinks)
    want = output64(q, k, v, mask)
    check_digits("o", _forward(q, k, v, mask, "kept"), *want)
    for mistake in ("none", "wrong"):
        got = _forward(q, k, v, mask, mistake)
        with pytest.raises(AssertionError, match="times its bound"):
            check_digits("o", got, *want)
        with pytest.raises(AssertionError, match="error of its rounding"):     # the norm by itself
            check_digits("o", got, want[0], torch.full_like(want[1], math.inf))
