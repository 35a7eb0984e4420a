"""Projections with 4-bit weights and group scales against 64-bit products, and their quantizer."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import runtime, torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def weights(g, n, k, group, scale):
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    scales = (0.001 + 0.01 * torch.rand(n, k // group, generator=g)).to(DT[scale])
    return q, scales


def dense(q, scales):
    """The weights as float64 [n][k]."""
    q = q.to(torch.int64)
    w = torch.stack([q & 15, q >> 4], dim=-1).view(q.shape[0], -1)
    w = torch.where(w > 7, w - 16, w).double()
    return w * scales.double().repeat_interleave(w.shape[1] // scales.shape[1], dim=1)


def reference(x, q, scales, act, residual=None):
    """float64 products and their error bound: x as integers of 2^-30 of its row's largest; float32 sums of
    k / 128 groups, 8 wavefronts and the digits and groups of a row (at most 16), over digits whose
    magnitudes exceed x's by less than 2^-5 of the largest; one rounding of the result."""
    w, xd = dense(q, scales), x.double()
    want = xd @ w.t()
    big = xd.abs().amax(dim=1, keepdim=True)
    tol = 2.0 ** -30 * big * w.abs().sum(1) + (w.shape[1] / 128 + 32) * 2.0 ** -24 * (
        (xd.abs() + 2.0 ** -5 * big) @ w.abs().t())
    if residual is not None:
        want = want + residual.double()
        tol = tol + 2.0 ** -24 * want.abs()
    return want, tol + STEP[act] * (want.abs() + tol) + TINY[act]


@pytest.mark.parametrize("act,scale,group,m,n,k", [
    ("f32", "f32", 32, 1, 1, 32), ("f32", "f16", 128, 1, 16, 128), ("f32", "f16", 64, 2, 17, 64),
    ("f32", "bf16", 32, 3, 100, 96), ("bf16", "bf16", 64, 5, 33, 320), ("f16", "f16", 128, 4, 50, 384),
    ("f32", "f16", 128, 1, 5632, 2048), ("bf16", "bf16", 32, 13, 2048, 5632), ("f16", "f32", 64, 16, 300, 2112),
    ("f32", "f32", 32, 8, 40, 8192), ("f32", "f16", 128, 33, 70, 1280), ("bf16", "f32", 64, 100, 31, 704),
    ("f32", "f32", 128, 1, 20, 131072), ("f16", "bf16", 32, 2, 9, 32768), ("f32", "f16", 128, 32, 64, 256),
    ("f32", "f16", 64, 7, 2000, 2048), ("f32", "f32", 128, 16, 8000, 2048), ("bf16", "f16", 32, 5, 20000, 512),
    ("f32", "bf16", 64, 4, 333, 4096), ("f32", "f16", 128, 3, 33, 16384), ("f16", "f16", 32, 6, 48, 16416),
    ("f32", "f16", 128, 1, 40, 16384), ("bf16", "f32", 64, 2, 40, 8192), ("f16", "f16", 32, 2, 24, 8224),
    ("f32", "bf16", 128, 1, 24, 16512), ("bf16", "f16", 64, 21, 50, 20480), ("f32", "f16", 32, 300, 70, 1056),
    ("bf16", "f16", 32, 1, 16400, 4096), ("f16", "f32", 32, 5, 16400, 2080),   # more scales than a first round of loads
])
def test_linear(serving, act, scale, group, m, n, k):
    """One row and many, widths and columns off the tiles, every group and type, strided rows, with and without a
    residual (also in place)."""
    g = torch.Generator().manual_seed(m * 7 + n + k)
    q, scales = weights(g, n, k, group, scale)
    lin = serving.W4Linear(q.cuda(), scales.cuda())
    wide = torch.randn(m, k + 24, generator=g)
    wide[:, 5::61] *= 30
    wide = wide.to(DT[act])
    x = wide[:, :k]
    want, tol = reference(x, q, scales, act)
    out = torch.full((m, n + 3), 6.0, dtype=DT[act], device="cuda")
    lin(wide.cuda()[:, :k], out=out[:, :n])
    worst = ((out[:, :n].cpu().double() - want).abs() / tol).max().item()
    assert worst <= 1, f"{worst} of the bound"
    assert (out[:, n:] == 6.0).all()
    res = torch.randn(m, n, generator=g).to(DT[act])
    want, tol = reference(x, q, scales, act, res)
    both = res.cuda()
    got = lin(x.contiguous().cuda(), residual=both)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    assert lin(x.contiguous().cuda(), residual=both, out=both) is both and torch.equal(both, got)


def test_exact_integers(serving):
    """Whole numbers and powers of two come out exactly: every nibble in every place, all digits of x, rows of
    very different and subnormal magnitudes, zeros."""
    n, k, group = 48, 512, 64
    g = torch.Generator().manual_seed(0)
    q = torch.arange(n * k // 2).remainder(256).to(torch.uint8).view(n, k // 2)
    scales = (2.0 ** torch.randint(-3, 4, (n, k // group), generator=g)).float()
    x = torch.zeros(9, k)
    x[0] = 1
    x[1, ::3] = -2.0 ** 100
    x[2, 1::5] = 2.0 ** -140
    x[3, 37] = 123456.0
    x[4, 100] = -(2.0 ** 23 + 1)
    x[5, 511] = 2.0 ** 127
    x[6, 0], x[6, 1] = 1.0, -2.0 ** -20
    x[8, 64:128] = torch.randint(-127, 128, (64,), generator=g).float()
    got = serving.W4Linear(q.cuda(), scales.cuda())(x.cuda()).cpu()
    want = x.double() @ dense(q, scales).t()
    assert torch.equal(got.double(), want.float().double())
    assert (got[7] == 0).all()


def test_range(serving):
    """Scales and rows near the ends of float32's range: results that fit are right, larger ones infinite, never
    not a number."""
    g = torch.Generator().manual_seed(9)
    q, _ = weights(g, 64, 256, 64, "f32")
    s = (2.0 ** torch.linspace(-125, 127, 64)).float()[:, None].expand(64, 4).contiguous()
    x = torch.randn(6, 256, generator=g) * torch.tensor([1, 1e30, 1e-30, 1e-8, 1e8, 2e-38])[:, None]
    got = serving.W4Linear(q.cuda(), s.cuda())(x.cuda()).cpu().double()
    want, tol = reference(x, q, s, "f32")
    # the sums are kept as y 2^(e - 52), 2^e times the row's largest in [2^29, 2^30): each of the 4 groups' additions
    # may lose 2^-150 there, up to 2^-150 2^52 max|x| / 2^29 = 2^-127 max|x| of y, for each of 4 digits
    tol = tol + 16 * 2.0 ** -127 * x.double().abs().amax(1, keepdim=True)
    big = want.abs() > 3.5e38
    assert not torch.isnan(got).any() and (got[big] == torch.sign(want[big]) * float("inf")).all()
    fits = want.abs() < 3.3e38
    assert ((got - want).abs() <= tol)[fits].all()


def test_special_values(serving):
    """An infinity or NaN makes its row NaN and no other; infinite and NaN scales reach their output."""
    g = torch.Generator().manual_seed(2)
    q, scales = weights(g, 40, 256, 128, "f32")
    x = torch.randn(4, 256, generator=g)
    clean = serving.W4Linear(q.cuda(), scales.cuda())(x.cuda())
    x[1, 200], x[3, 3] = float("inf"), float("nan")
    scales[7, 1] = float("nan")
    got = serving.W4Linear(q.cuda(), scales.cuda())(x.cuda())
    assert torch.isnan(got[[1, 3]]).all() and torch.isnan(got[:, 7]).all()
    keep = [i for i in range(40) if i != 7]
    assert torch.equal(got[[0, 2]][:, keep], clean[[0, 2]][:, keep])


@pytest.mark.parametrize("scale,group", [("f32", 32), ("bf16", 64), ("f16", 128)])
def test_quantizer(serving, scale, group):
    """Scales and weights are the formula's bits, groups of zeros and of numbers below the scales' range
    included."""
    g = torch.Generator().manual_seed(group)
    w = torch.randn(37, 3 * 128, generator=g) * torch.logspace(-4, 3, 37)[:, None]
    w[3, :group] = 0
    w[4, group:2 * group] = 1e-30
    w[5, 0] = 3e38
    got_q, got_s = serving.quantize_w4(w.cuda(), group, DT[scale])
    v = w.view(37, -1, group)
    s = (v.abs().amax(-1) / np.float32(7)).float()
    s = (s.clamp_max(65504.0) if scale == "f16" else s).to(DT[scale])
    zero = s == 0
    s = torch.where(zero, torch.ones_like(s), s)
    want = torch.where(zero[..., None], torch.zeros_like(v), (v / s.float()[..., None]).round().clamp(-8, 7))
    assert torch.equal(got_s.cpu(), s.view(37, -1))
    q = got_q.cpu().to(torch.int64)
    got = torch.stack([q & 15, q >> 4], -1).view(37, -1)
    got = torch.where(got > 7, got - 16, got)
    assert torch.equal(got, want.view(37, -1).to(torch.int64))
    x = torch.randn(3, 384, generator=g).cuda()
    same = serving.W4Linear.from_float(w.cuda(), group, DT[scale])(x)
    assert torch.equal(same, serving.W4Linear(got_q, got_s)(x))
    # within half a step of a weight, except where +-8 is clipped (the scales are rounded down)
    err = (dense(got_q.cpu(), got_s.cpu()).view_as(v) - v.double()).abs()
    inside = ~zero[..., None] & ((v / s.float()[..., None]).abs() <= 7.4)
    assert (err[inside] <= (0.5 + 1e-5) * s.double()[..., None].expand_as(err)[inside]).all()


def test_completing_form_and_graph(serving):
    """tl_linear_w4 gives the same bits; captured calls follow their inputs and share no scratch."""
    g = torch.Generator().manual_seed(5)
    q, scales = weights(g, 200, 1024, 64, "bf16")
    lin = serving.W4Linear(q.cuda(), scales.cuda())
    x = torch.randn(9, 1024, generator=g).cuda()
    want = lin(x)
    rt = runtime()
    y = torch.zeros_like(want)
    rt.call("tl_linear_w4", x, 1024, 0, 9, lin.packed, 1, 64, 200, 1024, None, 0, y, 200)
    assert torch.equal(y, want)
    rt.close()
    graphs = []
    for _ in range(2):
        xi = torch.randn(9, 1024, generator=g).cuda()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(lin(xi)[:, :8].repeat(1, 128).contiguous())
        graphs.append((graph, xi, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for _, xi, _ in graphs:
            xi.copy_(torch.randn(9, 1024, generator=g))
        torch.cuda.synchronize()
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, xi, out in graphs:
            assert torch.equal(out, lin(lin(xi)[:, :8].repeat(1, 128).contiguous()))


def test_refusals(serving):
    g = torch.Generator().manual_seed(1)
    q, scales = (t.cuda() for t in weights(g, 24, 256, 64, "f16"))
    lin = serving.W4Linear(q, scales)
    x = torch.zeros(2, 256, device="cuda")
    for bad in (lambda: serving.W4Linear(q.cpu(), scales), lambda: serving.W4Linear(q.int(), scales),
                lambda: serving.W4Linear(q[:, ::2], scales), lambda: serving.W4Linear(q, scales[:23]),
                lambda: serving.W4Linear(q, scales.double()), lambda: serving.W4Linear(q, scales[:, :1].contiguous()),
                lambda: serving.W4Linear(q, scales[:, :3].contiguous()), lambda: serving.W4Linear(q, scales[:, :0]),
                lambda: lin(x[:, :255]), lambda: lin(x.double()), lambda: lin(x.cpu()), lambda: lin(x[0]),
                lambda: lin(x, residual=torch.zeros(1, 24, device="cuda")), lambda: lin(x, out=torch.zeros(2, 23, device="cuda")),
                lambda: lin(x, residual=torch.zeros(2, 24, dtype=torch.float16, device="cuda")),
                lambda: lin(torch.zeros(2, 259, device="cuda")[:, 3:]), lambda: lin(x.t().contiguous().t()),
                lambda: serving.W4Linear.from_float(x, 48), lambda: serving.W4Linear.from_float(x.half()),
                lambda: serving.quantize_w4(x, 64, torch.float64), lambda: serving.quantize_w4(x.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    assert lin(x[:0]).shape == (0, 24)
