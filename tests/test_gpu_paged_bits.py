"""How many bits attention over the paged cache keeps of its probabilities."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu


def attend(act, cache, rows, heads, n, ones):
    """The operator's rows over one sequence of n keys with values in [1, 2) (or all 1), and the same in 64 bits."""
    from lpta import serving
    g = torch.Generator().manual_seed(1)
    page, hd = 16, 64
    pages = -(-n // page)
    shape = (pages, 1, page, hd)
    k = torch.randint(-127, 128, shape, generator=g).to(cache) if cache == torch.int8 else torch.randn(shape, generator=g).to(cache)
    v = torch.ones(shape).to(cache) if ones else (1 + torch.rand(shape, generator=g)).to(cache)
    scales = (torch.full((1,), 0.02), torch.ones(1)) if cache == torch.int8 else (None, None)
    q = torch.randn(rows, heads * hd, generator=g).to(act)
    c = serving.PagedCache(k.cuda(), v.cuda(), torch.arange(pages, dtype=torch.int32, device="cuda")[None],
                           *(None if s is None else s.cuda() for s in scales))
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    got = c.attend(q.cuda(), ids, ids + n - 1).cpu().view(rows, heads, hd)
    kd = k.double().view(-1, hd)[:n] * (1 if scales[0] is None else scales[0].double())
    p = torch.softmax(q.double().view(rows, heads, hd) @ kd.t() / 8, -1)
    return got, p @ v.double().view(-1, hd)[:n]


def test_bfloat16_probabilities_are_whole():
    """Results in [1, 2) have steps of 2^-7; one that is off by E is rounded to the wrong side where it lies within E of
    a middle, in 2 E / 2^-7 of all.  Over 2000 keys the scores' and exponentials' own errors average out to less than
    2^-20, so 2^-12 of the results may be wrong.  Two bfloat16 parts, truncated, would lose 2^-17.5 of every
    probability, the same way."""
    got, want = attend(torch.bfloat16, torch.bfloat16, 256, 8, 2000, False)
    wrong = int((got != want.to(torch.bfloat16)).sum())
    assert wrong <= got.numel() * 2.0 ** -12, wrong


@pytest.mark.parametrize("cache", [torch.float16, torch.int8, torch.bfloat16])
@pytest.mark.parametrize("ones", [True, False])
def test_float32_results_have_no_bias(cache, ones):
    """Each probability's parts, sum and quotient are rounded to nearest, so the mean over 512 rows and heads stays
    below half of float32's half step.  A truncated second float16 part loses 0.6 2^-23 on average, always downward."""
    got, want = attend(torch.float32, cache, 64, 8, 2000, ones)
    err = got.double() / want - 1
    assert err.mean().abs() <= 2.0 ** -25, err.mean().item()
    assert err.abs().max() <= 8 * 2.0 ** -24
