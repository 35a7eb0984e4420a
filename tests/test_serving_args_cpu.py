"""Arguments of the serving operators that are no tensors: wrong types are refused before anything is queued."""
import fractions

import numpy as np
import pytest
import torch

from lpta import serving
from lpta._native import TlPagedCache, TlValueError


def cache():
    """A cache's handle as the checks see it, its tensors in host memory, without a device's library."""
    c = object.__new__(serving.PagedCache)
    c.device, c.n_kv_heads, c.head_dim, c.n_seqs = torch.device("cpu"), 2, 64, 3
    c.desc = TlPagedCache(page_size=16, max_pages=8)
    c.rope = torch.zeros(128, 64), torch.zeros(128, 64)
    return c


def rows(n):
    return torch.zeros(0, n * 64), torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)


@pytest.mark.parametrize("prefix", [(0, 100.7), (0, 3.0), (0.5, 3), (1.0, 3), (0, "3"), (None, 3), (0, None), (0, float("nan")),
                                    (0, fractions.Fraction(7, 2)), (0, torch.tensor(3.5)), (0, [3])])
def test_a_prefix_is_whole_numbers(prefix):
    with pytest.raises(TlValueError, match="whole numbers"):
        cache().attend_shared(*rows(4), *prefix)


def test_prefixes_that_are():
    c = cache()
    for prefix in ((0, 3), (np.int64(2), np.int32(128)), (torch.tensor(1), torch.tensor(5)), (-7, 0), (99, 0), (True, True)):
        assert c.attend_shared(*rows(4), *prefix).shape == (0, 256)
    for prefix in ((0, -1), (0, 129), (3, 1), (-1, 1), (0, 1 << 70)):
        with pytest.raises(TlValueError, match="pages of a sequence"):
            c.attend_shared(*rows(4), *prefix)


def test_norms():
    c = cache()
    gain = torch.ones(64)
    for norm in ((gain, gain), [None, gain], (gain, None), torch.ones(2, 64), (None, None)):
        for eps in (0, 0.0, 1e-6, np.float32(1e-5), 1e30):
            assert c.append(*rows(8), norm=norm, eps=eps).shape == (0, 256)
    for norm in (5, gain, (gain,), (gain, gain, gain), (gain, 1.0), (gain, gain[:32]), (gain.double(), gain), "qk", torch.tensor(1.0),
                 (torch.ones(128)[::2], gain), {"q": gain, "k": gain}):
        with pytest.raises(TlValueError):
            c.append(*rows(8), norm=norm)
    for eps in (-1e-9, float("nan"), float("inf"), 2e30, "1e-5", None, torch.tensor(1e-5), 1j):
        with pytest.raises(TlValueError, match="eps"):
            c.append(*rows(8), norm=(gain, gain), eps=eps)
