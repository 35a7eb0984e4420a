"""A handle of another device is refused wherever one can be given, before anything is queued."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu


class OtherDevice:
    """A handle of a device that the tensors are not on; it takes no calls."""
    device = 7


def test_a_handle_of_another_device():
    from lpta import serving
    rt = OtherDevice()
    w = torch.randn(16, 64, device="cuda")
    q, scales = serving.quantize_w4(w, 32)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device="cuda")
    ids = torch.zeros(16, dtype=torch.int32, device="cuda")
    for call in (lambda: serving.quantize_w4(w, 32, rt=rt), lambda: serving.W4Linear.from_float(w, 32, rt=rt),
                 lambda: serving.W4Linear(q, scales, rt=rt), lambda: serving.token_logprobs(w, ids, rt=rt),
                 lambda: serving.PagedCache(k, k.clone(), ids[None, :1], rt=rt)):
        with pytest.raises(ValueError, match="another device"):
            call()
