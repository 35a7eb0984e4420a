"""What the serving operators' header says of numbers that are not finite, where the operators' own tests say nothing."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch
from test_gpu_w4 import weights

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k", [(1, 256), (4, 256), (13, 1024), (2, 20480)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_scales_that_are_not_finite(m, k, bad):
    """Each leaves its column infinite or NaN (digits of zero times infinity are NaN) and no other."""
    from lpta import serving
    g = torch.Generator().manual_seed(m)
    q, scales = weights(g, 40, k, 128, "f32")
    x = torch.randn(m, k, generator=g)
    x[0, :128] = 0
    clean = serving.W4Linear(q.cuda(), scales.cuda())(x.cuda())
    scales[7, 1] = scales[22, 0] = bad
    got = serving.W4Linear(q.cuda(), scales.cuda())(x.cuda())
    keep = [n for n in range(40) if n not in (7, 22)]
    assert not torch.isfinite(got[:, [7, 22]]).any() and torch.equal(got[:, keep], clean[:, keep])


@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
def test_a_key_that_is_not_finite(cache):
    """It reaches the rows that attend it and the heads of its KV head, and no others."""
    from lpta import serving
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(20, 2, 16, 64, generator=g).to(cache).cuda() for _ in range(2))
    c = serving.PagedCache(k, v, torch.arange(20, dtype=torch.int32, device="cuda")[None])
    pos = torch.tensor([319, 100, 99, 40], dtype=torch.int32, device="cuda")
    seq = torch.zeros(4, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 8 * 64, generator=g).cuda()
    clean = c.attend(q, seq, pos)
    for bad in (float("inf"), -float("inf"), float("nan")):
        k[6, 1, 4, 3] = bad                       # position 100 of KV head 1
        got = c.attend(q, seq, pos)
        assert torch.equal(got[2:], clean[2:]) and torch.equal(got[:2, :256], clean[:2, :256])
        if bad != bad:
            assert torch.isnan(got[:2, 256:]).all()
