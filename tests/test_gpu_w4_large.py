"""The 4-bit quantizer past the weights that one launch's threads take."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu


def test_quantizer_past_one_launch():
    """2^24 x 1056 weights, 71 GB: rows at the start, around the first pass's end and last are those of a small matrix."""
    from lpta import serving
    n, k, group = 1 << 24, 1056, 32
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip("needs 110 GiB of free GPU memory")
    at = torch.tensor([0, 1, 2 ** 34 // k - 1, 2 ** 34 // k, 2 ** 34 // k + 1, n - 2, n - 1], device="cuda")
    some = torch.randn(len(at), k, generator=torch.Generator().manual_seed(1)).cuda()
    w = torch.zeros(n, k, device="cuda")
    w[at] = some
    q, scales = serving.quantize_w4(w, group)
    del w
    want_q, want_s = serving.quantize_w4(some, group)
    assert torch.equal(q[at], want_q) and torch.equal(scales[at], want_s)
    q[at], scales[at] = 0, 1
    assert not q.any() and (scales == 1).all()
    del q, scales
    torch.cuda.empty_cache()
