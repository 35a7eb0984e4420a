"""Projections with 8-bit weights and rows, alone and gated, against the definition in 64 bits."""
from __future__ import annotations

import pytest

from gpu_util import runtime, torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# a rounding is off by at most half a step: eps / 2, or half the least subnormal number
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def quantized(x):
    """q (float64 integers) and s of each row: s = f32(max / 127), q = clip(rne(f32(x / s))); a float64 quotient of
    two float32 numbers rounds to their float32 quotient."""
    x = x.double()
    s = (x.abs().amax(dim=1) / 127).float().double()
    s[s == 0] = 1
    return torch.round((x / s[:, None]).float()).clamp(-127, 127).double(), s


def product(x, w, scales):
    """float64 results and their float32 error bound: the sum's conversion, s_m s_n and their product round."""
    q, s = quantized(x)
    y = (q @ w.double().t()) * s[:, None] * scales.double()
    return y, 3.01 * U * y.abs() + 2.0 ** -149


def close(got, want, tol, act):
    # half a step of the type at most from what lies tol from the value
    bound = tol + STEP[act] * (want.abs() + tol) + TINY[act]
    if want.numel():
        worst = ((got.cpu().double() - want).abs() / bound).max().item()
        assert worst <= 1, f"{worst} of the bound"


def weights(g, n, k):
    return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g) * 1e-3 + 1e-5


SHAPES = [
    # act, m, n, k, residual
    ("f32", 1, 1, 1, False), ("f32", 1, 16, 64, True), ("f32", 1, 2048, 5632, True), ("bf16", 1, 5632, 2048, False),
    ("f16", 2, 33, 77, True), ("f32", 3, 300, 1001, False), ("bf16", 4, 200, 8192, False), ("f32", 4, 17, 8191, True),
    ("f32", 1, 40, 32768, False), ("f16", 1, 40, 32769, False),               # around the rows a thread keeps
    ("bf16", 2, 100, 20000, True), ("f32", 5, 64, 128, False), ("f32", 16, 100, 300, True), ("bf16", 17, 48, 129, False),
    ("f32", 32, 500, 640, True), ("f16", 33, 1000, 200, False), ("bf16", 45, 6144, 4096, False), ("f32", 64, 40, 65, False),
    ("bf16", 65, 130, 1000, True), ("f32", 255, 257, 383, False), ("f16", 256, 64, 96, True), ("f32", 257, 129, 127, True),
    ("bf16", 300, 127, 2049, False), ("f16", 513, 1000, 640, True), ("f32", 700, 2050, 513, False),
    ("bf16", 2000, 6200, 300, True), ("f32", 1000, 14000, 200, False), ("f16", 4097, 4097, 130, False),
    ("f32", 5, 20, 131072, False), ("f32", 300, 20, 131072, False),           # the longest sums
    ("f32", 9000, 16, 64, False),
]


@pytest.mark.parametrize("act,m,n,k,residual", SHAPES)
def test_linear(serving, act, m, n, k, residual):
    g = torch.Generator().manual_seed(m + n + k)
    w, s = weights(g, n, k)
    x = torch.randn(m, k, generator=g)
    x[:, ::53] *= 9
    x *= torch.exp(2 * torch.randn(m, 1, generator=g))
    x = x.to(DT[act])
    r = torch.randn(m, n, generator=g).to(DT[act]) if residual else None
    lin = serving.W8Linear(w.cuda(), s.cuda())
    y = lin(x.cuda(), residual=None if r is None else r.cuda())
    assert y.dtype == DT[act] and y.shape == (m, n)
    want, tol = product(x, w, s)
    if residual:
        want = want + r.double()
        tol = tol + U * (want.abs() + tol)
    close(y, want, tol, act)


def silu_bound(gate, tg, up, tu):
    """silu(g) u and its bound: silu's slope is at most 1.1 and at most (1 + |g|) |silu| / |g| from 0 down, so an error
    tg moves it by min(1.1 tg, (1 + |g|) tg |silu| / |g|) ; the exponential (3 2^-24 and its argument's rounding,
    2^-24 |g| at most), the sum, the quotient and two products, 2^-24 each, of itself.  Below -80 it is taken as 0."""
    silu = torch.nn.functional.silu(gate)
    slope = torch.where(gate > 0, 1.1, torch.minimum(torch.full_like(gate, 1.1), (1 + gate.abs()) * silu.abs() / gate.abs().clamp_min(1e-300) * 1.001))
    ts = slope * tg + (8 + gate.abs().clamp_max(80)) * U * silu.abs() + torch.where(gate < -79.9, 2e-33, 0.0) + 2.0 ** -149
    return silu * up, ts * up.abs() + (silu.abs() + ts) * tu + U * (silu * up).abs()


@pytest.mark.parametrize("act,m,n,k", [
    ("f32", 1, 1, 1), ("f32", 1, 5632, 2048), ("bf16", 2, 40, 333), ("f16", 4, 100, 4096), ("f32", 7, 33, 129),
    ("bf16", 16, 5632, 512), ("f32", 32, 1000, 2048), ("f16", 40, 65, 1000), ("f32", 200, 130, 257), ("bf16", 256, 31, 640),
    ("f32", 258, 40, 200), ("bf16", 600, 1111, 385), ("f16", 2001, 3000, 256), ("f32", 1, 100, 40000)])
def test_gated(serving, act, m, n, k):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    (w, s), (w2, s2) = weights(g, n, k), weights(g, n, k)
    x = (torch.randn(m, k, generator=g) * torch.exp(1.5 * torch.randn(m, 1, generator=g)) * 0.3).to(DT[act])
    y = serving.W8GatedLinear(w.cuda(), s.cuda(), w2.cuda(), s2.cuda())(x.cuda())
    want, tol = silu_bound(*product(x, w, s), *product(x, w2, s2))
    # what float16 cannot hold is infinite on both sides
    if act == "f16":
        big = want.abs() > 65000
        want, tol, y = want.masked_fill(big, 0), tol.masked_fill(big, 0), y.cpu().masked_fill(big, 0)
    close(y, want, tol, act)


def test_silu_far_out(serving):
    """Gates from -3e38 to 3e38, zeros among them."""
    x = torch.tensor([[1.0]], device="cuda")
    gates = torch.tensor([-3e38, -1e6, -200, -89, -80.5, -80.0, -79, -60, -30, -20, -1, -1e-3, -1e-30, 0, 1e-30, 1e-3, 1, 20, 60, 80,
                          100, 1e6, 3e38])
    w = torch.full((len(gates), 1), 127, dtype=torch.int8, device="cuda")
    s = (gates / 127).cuda()
    one = torch.full((len(gates),), 1 / 127, device="cuda")
    # x = 1: q = 127 and s_x = 1 / 127, so that the gate is 127 * 127 / 127 s_n
    y = serving.W8GatedLinear(w, s, w, one)(x)
    gate = 127 * 127 * torch.tensor(1 / 127).double() * s.cpu().double()
    up = 127 * 127 * torch.tensor(1 / 127).double() ** 2
    want, tol = silu_bound(gate[None], 3.01 * U * gate[None].abs() + 2.0 ** -149, up.expand(1, len(gates)),
                           3.01 * U * up.expand(1, len(gates)))
    close(y, want, tol, "f32")


def test_exact_integers(serving):
    """Sums past 2^24 and near 2^31 are exact: rows whose scale is 1, weights' scale a power of two."""
    k = 131072
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 5
    x = torch.full((6, k), 127.0)
    x[1, 1::3] = -127
    x[2, 7] = -3
    s = torch.full((3,), 0.5)
    for rows in (1, 6):
        y = serving.W8Linear(w.cuda(), s.cuda())(x[:rows].cuda())
        want = (x[:rows].double() @ w.double().t() * 0.5).float()   # rounded once, as the conversion does
        assert torch.equal(y.cpu(), want)


def test_rounding_of_rows(serving):
    """Quotients half way between integers go to the even one, in every kernel that quantizes."""
    k = 254
    x = torch.arange(-127, 127).float() + 0.5
    x[0], x[-1] = -127, 127
    w = torch.eye(k, dtype=torch.int8)
    for m in (1, 3, 20, 300):
        y = serving.W8Linear(w.cuda(), torch.ones(k).cuda())(x.expand(m, k).contiguous().cuda())
        assert torch.equal(y.cpu(), torch.round(x).expand(m, k))


@pytest.mark.parametrize("m", [1, 4, 9, 70, 300])
def test_special_rows(serving, m):
    """Rows of zeros give zeros (and the residual), an infinity or NaN its own row of NaN and no other; tiny and huge rows."""
    g = torch.Generator().manual_seed(m)
    w, s = weights(g, 70, 200)
    lin = serving.W8Linear(w.cuda(), s.cuda())
    pair = serving.W8GatedLinear(w.cuda(), s.cuda(), w.cuda(), s.cuda())
    for bad in (float("nan"), float("inf"), -float("inf"), 0.0, 1e-42, 1e-30, 3e38):
        x = torch.randn(m, 200, generator=g)
        row = m // 2
        if bad == 0.0:
            x[row] = 0
        elif abs(bad) < 1 or bad == 3e38:
            x[row] *= bad / x[row].abs().max()
        else:
            x[row, 199] = bad
        y, z = lin(x.cuda()), pair(x.cuda())
        others = [i for i in range(m) if i != row]
        want, tol = product(x[others], w, s)
        close(y[others], want, tol, "f32")
        if bad == 0.0:
            assert (y[row] == 0).all() and (z[row] == 0).all()
        elif bad in (float("inf"), -float("inf")) or bad != bad:
            assert torch.isnan(y[row]).all() and torch.isnan(z[row]).all() and torch.isfinite(z[others]).all()
        else:
            want, tol = product(x[row:row + 1], w, s)
            close(y[row:row + 1], want, tol, "f32")


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(1, 70, 203), (3, 65, 130), (20, 67, 203), (300, 131, 140), (600, 2049, 141)])
def test_strides(serving, act, m, n, k):
    """Rows of any stride and alignment; what lies between and behind them stays; out is the residual."""
    g = torch.Generator().manual_seed(n)
    w, s = weights(g, n, k)
    lin = serving.W8Linear(w.cuda(), s.cuda())
    for pad, off in ((1, 1), (8, 0), (3, 2)):
        wide = torch.randn(m, k + pad + off, generator=g).to(DT[act]).cuda()
        x = wide[:, off:off + k]
        buf = torch.full((m + 1, n + pad + off), 7.0, dtype=DT[act], device="cuda")
        y = buf[:m, off:off + n]
        lin(x, out=y)
        plain = lin(x.contiguous())
        assert torch.equal(y, plain)
        rest = buf.clone()
        rest[:m, off:off + n] = 7.0
        assert (rest == 7.0).all()
        lin(x, residual=y, out=y)
        assert torch.equal(y, lin(x.contiguous(), residual=plain))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2, 40, 64), (20, 100, 200), (200, 130, 70),       # registers, K split
                                   (513, 4000, 64), (1000, 14000, 40), (1000, 14001, 130),   # tiles of 8 x 8, 14 x 16
                                   (1100, 9000, 64), (256, 65536, 40)])               # 16 x 14, 16 x 16
def test_out_is_residual(serving, act, m, n, k):
    """Every result takes its residual once, where it is written over it too."""
    g = torch.Generator().manual_seed(m + n)
    w, s = weights(g, n, k)
    lin = serving.W8Linear(w.cuda(), s.cuda())
    x = torch.randn(m, k, generator=g).to(DT[act]).cuda()
    r = torch.randn(m, n, generator=g).to(DT[act]).cuda()
    want = lin(x, residual=r)
    for _ in range(2):
        y = r.clone()
        assert lin(x, residual=y, out=y) is y
        assert torch.equal(y, want)


def test_packing_of_few_columns_and_quantizer(serving):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(50, 70, generator=g)
    w[4] = 0
    q, s = serving.quantize_w8(w.cuda())
    assert (q[4] == 0).all() and s[4] == 1
    want = w.abs().amax(dim=1) / 127
    want[4] = 1
    assert torch.equal(s.cpu(), want)
    assert torch.equal(q.cpu(), torch.round((w.double() / want.double()[:, None]).float()).clamp(-127, 127).to(torch.int8))
    x = torch.randn(6, 70, generator=g).cuda()
    assert torch.equal(serving.W8Linear(q, s)(x), serving.W8Linear.from_float(w.cuda())(x))
    assert torch.equal(serving.W8GatedLinear(q, s, q, s)(x), serving.W8GatedLinear.from_float(w.cuda(), w.cuda())(x))


def test_completing_form_graph_and_streams(serving):
    """The completing entry point, calls captured and replayed beside eager ones, calls on streams of their own."""
    g = torch.Generator().manual_seed(8)
    w, s = weights(g, 200, 640)
    lin = serving.W8Linear(w.cuda(), s.cuda())
    sizes = (1, 30, 300)
    xs = [torch.randn(m, 640, generator=g).cuda() for m in sizes]
    want = [lin(x) for x in xs]
    torch.cuda.synchronize()
    rt = runtime()
    for x, y in zip(xs, want):
        out = torch.empty_like(y)
        rt.call("tl_linear_w8", x, 640, 0, len(x), lin.packed, 0, 200, 640, None, 0, out, 200)
        assert torch.equal(out, y)
    rt.close()
    graphs = []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(x)
        graphs.append((graph, x, out))
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(4):
        for graph, x, out in graphs:
            x.copy_(torch.randn(x.shape, generator=g))
            out.zero_()
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [lin(x) for _, x, _ in graphs]
        torch.cuda.synchronize()
        for (_, _, out), y in zip(graphs, eager):
            assert torch.equal(out, y)


def test_refusals(serving):
    w, s = weights(torch.Generator().manual_seed(1), 32, 48)
    w, s = w.cuda(), s.cuda()
    lin, pair = serving.W8Linear(w, s), serving.W8GatedLinear(w, s, w, s)
    x = torch.randn(4, 48, device="cuda")
    y = torch.randn(4, 32, device="cuda")

    class Other:
        device = 7
    for bad in (lambda: lin(x.double()), lambda: lin(x.cpu()), lambda: lin(x[:, :40]), lambda: lin(x[0]), lambda: lin(x.t()),
                lambda: lin(x, residual=y[:3]), lambda: lin(x, residual=y.half()), lambda: lin(x, out=y[:, :30]),
                lambda: lin(x, out=y.bfloat16()), lambda: lin(x, out=y[:3]), lambda: lin(x[:, :1].expand(4, 48)),
                lambda: lin(x[:1].expand(4, 48)), lambda: lin(x, out=x[:, :32]), lambda: pair(x, out=x[:, :32]),
                lambda: lin(x, residual=y, out=y[:, :32].t().contiguous().t()),
                lambda: serving.W8Linear(w.cpu(), s), lambda: serving.W8Linear(w.float(), s), lambda: serving.W8Linear(w.t(), s),
                lambda: serving.W8Linear(w, s[:30]), lambda: serving.W8Linear(w, s.double()), lambda: serving.W8Linear(w, s.cpu()),
                lambda: serving.W8Linear(w[0], s), lambda: serving.W8Linear(w[:0], s[:0]), lambda: serving.W8Linear(w[:, :0], s),
                lambda: serving.W8GatedLinear(w, s, w[:16].contiguous(), s[:16]), lambda: serving.W8GatedLinear(w, s, w, s[:16]),
                lambda: serving.W8Linear(w, s, rt=Other()), lambda: serving.quantize_w8(w), lambda: serving.quantize_w8(x.cpu()),
                lambda: serving.quantize_w8(x[0]), lambda: serving.quantize_w8(x[:0]), lambda: serving.quantize_w8(x, rt=Other())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="2\\^17"):
        serving.W8Linear(torch.zeros(1, (1 << 17) + 1, dtype=torch.int8, device="cuda"), s[:1])
    assert lin(x[:0]).shape == (0, 32) and pair(x[:0]).shape == (0, 32)
