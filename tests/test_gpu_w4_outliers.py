"""4-bit projections of rows with outliers: what a far larger value leaves of the others."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch
from test_gpu_w4 import STEP, DT, dense, weights

torch = get_torch()
pytestmark = pytest.mark.gpu


def bound(x, w, y, act):
    """A value is off by half of 2^-29 of the largest of its 128 columns; then float32 sums of k / 128 blocks (up to 4
    groups in each), 8 wavefronts and the digits of a row, over digits whose magnitudes exceed x's by less than 2^-5 of
    the block's largest; one rounding."""
    m, k = x.shape
    pad = -k % 128
    xb = torch.nn.functional.pad(x.abs(), (0, pad)).view(m, -1, 128)
    wb = torch.nn.functional.pad(w.abs(), (0, pad)).view(w.shape[0], -1, 128)
    most = xb.amax(2)
    fixed = 2.0 ** -30 * (most @ wb.sum(2).t())
    sums = (4 * (k / 128) + 16) * 2.0 ** -24 * (x.abs() @ w.abs().t() + 2.0 ** -5 * (most @ wb.sum(2).t()))
    return fixed + sums + STEP[act] * (y.abs() + fixed + sums)


# up to four rows in one kernel, more in two, rows longer than a workgroup's registers
@pytest.mark.parametrize("m,n,k,group", [(1, 300, 2048, 128), (2, 64, 4096, 64), (4, 100, 1056, 32), (9, 5632, 1024, 64),
                                         (16, 300, 4096, 128), (2, 40, 20480, 32), (21, 48, 20480, 128), (5, 33, 32, 32)])
def test_outliers_leave_other_columns_their_bits(m, n, k, group):
    """An outlier whose block of 128 columns has no weights: float32's bound for all other columns, whatever its size.
    (Where a row is one block there are no others, and the result is zero.)"""
    from lpta import serving
    g = torch.Generator().manual_seed(m + k)
    q, scales = weights(g, n, k, group, "f32")
    at = (k // 2) // 128 * 128
    q[:, at // 2:(at + 128) // 2] = 0
    lin = serving.W4Linear(q.cuda(), scales.cuda())
    w = dense(q, scales)
    for size in (3e3, 3e6, 2.0 ** 40, 2.0 ** 120):
        x = torch.randn(m, k, generator=g)
        x[:, min(at + 77, k - 1)] = size
        want = x.double() @ w.t()
        got = lin(x.cuda()).cpu().double()
        # 64 bits more than the outlier's are kept: below that, 2^-94 of it
        tol = bound(x.double().where(x < size, 0.0), w, want, "f32") + 2.0 ** -94 * size * w.abs().sum(1)
        assert ((got - want).abs() <= tol).all(), (size, ((got - want).abs() / tol).max().item())


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
def test_an_outlier_beside_small_values(act):
    """One value of 3000 times the rest whose own weight is zero: with the error of a block's fixed point the result
    stays inside what float32 sums alone may lose."""
    from lpta import serving
    g = torch.Generator().manual_seed(3)
    n, k = 256, 4096
    q, scales = weights(g, n, k, 128, "f32")
    q[:, 1000 // 2] &= 0xF0
    lin = serving.W4Linear(q.cuda(), scales.cuda())
    w = dense(q, scales)
    for m in (1, 3, 11):
        x = torch.randn(m, k, generator=g)
        x[:, 1000] = 3000
        x = x.to(DT[act])
        want = x.double() @ w.t()
        got = lin(x.cuda()).cpu().double()
        tol = k * 2.0 ** -24 * (x.double().abs() @ w.abs().t())
        rms = ((got - want) ** 2).mean().sqrt() / (want ** 2).mean().sqrt()
        assert ((got - want).abs() <= tol + STEP[act] * want.abs()).all()
        assert act != "f32" or rms <= 2.0 ** -21.5, rms.item()   # 3.4e-7: rms over 32 blocks' fixed point and sums


def test_blocks_of_very_different_sizes():
    """Blocks of powers of two from one end of float32 to the other, alone and together, exactly."""
    from lpta import serving
    g = torch.Generator().manual_seed(4)
    k = 2048
    q = torch.randint(0, 256, (32, k // 2), dtype=torch.uint8, generator=g)
    lin = serving.W4Linear(q.cuda(), torch.ones(32, k // 64).cuda())
    w = dense(q, torch.ones(32, k // 64))
    x = torch.zeros(7, k)
    for b in range(16):
        x[b % 4, b * 128 + 3 * b] = 2.0 ** (-120 + 15 * b)     # sums of four that lie 60 bits apart
        x[4, b * 128 + 5] = 2.0 ** (b - 8)
        x[5, b * 128 + 9] = 2.0 ** -140
    x[6, :128] = 1e-30
    x[6, 200] = 1e30
    got = lin(x.cuda()).cpu().double()
    want = x.double() @ w.t()
    # a partial sum is below 8 2^127 2^-52 of the frame it is kept in, whose steps end at 2^-149
    big = x.double().abs().amax(1, keepdim=True)
    tol = 4 * 2.0 ** -24 * want.abs() + 2.0 ** -90 * big
    assert torch.equal(got[4:6], want[4:6]) and ((got - want).abs() <= tol).all()
