"""Alternatives of rows with few numbers among NaN, in parts that do not fill the kernel's tiles."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(100, 17000), (130, 9000), (128, 12281), (130, 8186), (90, 18425), (300, 16385)])
def test_few_numbers_among_nan(dtype, rows, vocab):
    """Rows of NaN, with one number, and with some numbers and minus infinities in every part: NaN are never named, -1
    where too few are left; the rows beside them as ever."""
    from lpta import serving
    top = 11
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x[::3] = np.nan
    x[3, vocab // 2] = 0.5
    for r in range(6, rows, 6):
        at = rng.choice(vocab, r % 17, replace=False)
        x[r, at] = rng.standard_normal(len(at))
        x[r, at[::3]] = -np.inf
    x[9, ::500] = -np.inf
    t = torch.from_numpy(x).to(getattr(torch, dtype))
    got = serving.token_logprobs(t.cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda"), top)
    ids, tops, lp = (v.cpu().numpy() for v in (got.top_ids, got.top_logprobs, got.logprob))
    x = t.float().numpy()
    for r in range(rows):
        numbers = np.flatnonzero(~np.isnan(x[r]))
        want = numbers[np.lexsort((numbers, -x[r, numbers]))][:top]
        assert ids[r].tolist() == want.tolist() + [-1] * (top - len(want)), r
        assert np.isnan(tops[r]).all() == (r % 3 == 0) and np.isnan(lp[r]) == (r % 3 == 0)
