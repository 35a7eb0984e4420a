"""8-bit projections against the definition in 64 bits at the sizes that take every way through their kernels."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch
from test_gpu_w8 import DT, STEP, TINY, U, product, silu_bound
from w8_paths import PAST_ROWS, ROW_CASES, TILE_CASES

torch = get_torch()
pytestmark = pytest.mark.gpu


def near(got, want, tol, act):
    """Half a step of the type at most from what lies tol from the value; what float16 cannot hold is infinite."""
    bound = tol + STEP[act] * (want.abs() + tol) + TINY[act]
    off = (got.double() - want).abs()
    if act == "f16":
        off = off.masked_fill(want.abs() > 65000, 0)
    worst = (off / bound).max().item()
    assert worst <= 1, f"{worst} of the bound"


@pytest.mark.parametrize("m,n,k,gated", TILE_CASES + ROW_CASES + PAST_ROWS)
def test_every_way(m, n, k, gated):
    from lpta import serving
    act = ("f32", "bf16", "f16")[(m + k) % 3]
    g = torch.Generator("cuda").manual_seed(m + 3 * n + 5 * k)
    pairs = [(torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device="cuda"),
              torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-5) for _ in range(1 + gated)]
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    x[:, ::53] *= 5
    x = (x * (0.3 if gated else 1.0)).to(DT[act])
    if gated:
        y = serving.W8GatedLinear(*pairs[0], *pairs[1])(x)
        # sums of whole numbers below 2^53 are exact in 64 bits, in any order
        want, tol = silu_bound(*product(x, *pairs[0]), *product(x, *pairs[1]))
    else:
        r = torch.randn(m, n, generator=g, device="cuda").to(DT[act]) if k % 2 else None
        y = serving.W8Linear(*pairs[0])(x, residual=r)
        want, tol = product(x, *pairs[0])
        if r is not None:
            want = want + r.double()
            tol = tol + U * (want.abs() + tol)
    assert y.dtype == DT[act] and y.shape == (m, n)
    near(y, want, tol, act)
