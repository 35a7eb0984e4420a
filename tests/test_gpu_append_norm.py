"""The append with norms of q and k for each head, against its definition."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import runtime, torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def tables(n, hd):
    inv = 10000.0 ** (-np.arange(0, hd, 2) / hd)
    a = np.concatenate([np.arange(n)[:, None] * inv] * 2, axis=1)
    return torch.from_numpy(np.cos(a).astype(np.float32)), torch.from_numpy(np.sin(a).astype(np.float32))


def normed(x, gain, eps):
    """x [..., hd] float32 to x f gain, the factor in 64 bits and rounded once, the products float32."""
    if gain is None:
        return x
    f = (1 / np.sqrt((x.astype(np.float64) ** 2).mean(axis=-1, keepdims=True) + eps)).astype(np.float32)
    return (x * f) * gain


def rotated(x, cos, sin):
    h = x.shape[-1] // 2
    turned = np.concatenate([-x[..., h:], x[..., :h]], axis=-1)
    return x * cos[:, None] + turned * sin[:, None]


def rows_of(cache, which, table, seq, pos, page):
    """The cache's row of each (sequence, position), [n][kv][hd]."""
    return torch.stack([which[int(table[s, p // page]), :, p % page] for s, p in zip(seq, pos)])


CASES = [("f32", "i8", 8, 2, 64, 16, 1), ("f32", "i8", 32, 4, 64, 8, 37), ("bf16", "bf16", 32, 8, 128, 16, 75),
         ("f16", "f16", 5, 5, 128, 64, 300), ("f32", "f16", 1, 1, 128, 32, 9), ("bf16", "i8", 12, 12, 64, 128, 20),
         ("f16", "bf16", 7, 1, 64, 1024, 130), ("f32", "bf16", 40, 8, 128, 16, 3), ("f32", "i8", 0, 3, 64, 16, 11)]


@pytest.mark.parametrize("act,cache,heads,kv,hd,page,rows", CASES)
@pytest.mark.parametrize("which", ["both", "q", "k"])
def test_append_norm(serving, act, cache, heads, kv, hd, page, rows, which):
    """q, k and v of ragged rows, a padded row and a row in place among them: the INT8 and 16-bit rows are the
    definition's steps bit for bit, and float results within their roundings of the 64-bit value."""
    g = torch.Generator().manual_seed(rows + heads)
    seqs = min(rows, 5)
    pos = [(i // seqs) * 3 + i % 3 for i in range(rows)]
    seq = [i % seqs for i in range(rows)]
    if rows > 2:
        seq[2] = -1
    cols = max(pos) // page + 1
    table = torch.randperm(seqs * cols + 2, generator=g)[:seqs * cols].view(seqs, cols).to(torch.int32)
    cos, sin = tables(max(pos) + 1, hd)
    x = torch.randn(rows, heads + 2 * kv, hd, generator=g) * torch.exp(2 * torch.randn(rows, heads + 2 * kv, 1, generator=g))
    x = x.to(DT[act])
    gains = [1 + 0.4 * torch.randn(hd, generator=g) for _ in range(2)]
    q_gain, k_gain = gains[0] if which != "k" else None, gains[1] if which != "q" else None
    scales = [0.03 + 0.02 * torch.rand(kv, generator=g) for _ in range(2)] if cache == "i8" else [None, None]
    pool = [torch.zeros(seqs * cols + 2, kv, page, hd, dtype=DT[cache], device="cuda") for _ in range(2)]
    c = serving.PagedCache(*pool, table.cuda(), *(None if s is None else s.cuda() for s in scales), rope=(cos.cuda(), sin.cuda()))
    ids = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (seq, pos)]
    norm = tuple(None if t is None else t.cuda() for t in (q_gain, k_gain))
    flat = x.view(rows, -1).cuda()
    out = torch.full((rows, heads * hd), 9.0, dtype=DT[act], device="cuda")
    eps = 1e-6
    c.append(flat, *ids, out=out, norm=norm, eps=eps)
    c.check()
    xf = x.float().numpy()
    cs, sn = cos.numpy()[pos], sin.numpy()[pos]
    gn = [None if t is None else t.numpy() for t in (q_gain, k_gain)]
    live = [i for i in range(rows) if seq[i] >= 0]
    want_q = torch.from_numpy(rotated(normed(xf[:, :heads], gn[0], eps), cs, sn)).to(DT[act]).reshape(rows, -1)
    assert torch.equal(out.cpu()[live], want_q[live])
    for i in range(rows):
        if seq[i] < 0:
            assert (out[i] == 9.0).all()
    want_k = torch.from_numpy(rotated(normed(xf[:, heads:heads + kv], gn[1], eps), cs, sn))
    want_v = torch.from_numpy(xf[:, heads + kv:])
    for t, want, s in ((c.k, want_k, scales[0]), (c.v, want_v, scales[1])):
        if cache == "i8":
            want = torch.round(want / s[:, None]).clamp(-127, 127)
        got = rows_of(c, t.cpu(), table, [seq[i] for i in live], [pos[i] for i in live], page)
        assert torch.equal(got, want[live].to(DT[cache]))
    # against 64 bits: the factor, three products and a sum round to float32, then the result to its type
    xd = x.double()[:, :heads]
    if q_gain is not None:
        xd = xd / (xd.pow(2).mean(dim=-1, keepdim=True) + eps).sqrt() * q_gain.double()
    h = hd // 2
    turned = torch.cat([-xd[..., h:], xd[..., :h]], dim=-1)
    cd, sd = (torch.from_numpy(t).double()[:, None] for t in (cs, sn))
    want = (xd * cd + turned * sd).reshape(rows, -1)
    mag = ((xd * cd).abs() + (turned * sd).abs()).reshape(rows, -1)
    tol = 5.1 * 2.0 ** -24 * mag + 2.0 ** -148
    tol = tol + STEP[act] * (want.abs() + tol) + TINY[act]
    assert ((out.cpu().double() - want).abs() <= tol)[live].all()
    if heads and rows > 1:   # in place
        before = flat.clone()
        c.append(flat, *ids, out=flat[:, :heads * hd], norm=norm, eps=eps)
        assert torch.equal(flat[live, :heads * hd], out[live])
        assert torch.equal(flat[:, heads * hd:], before[:, heads * hd:])


def test_zeros_and_extremes(serving):
    """A head of zeros is zeros; values whose squares leave float32's range are normed; without eps zeros are NaN; an
    infinity stays in its head."""
    cos, sin = tables(4, 64)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device="cuda")
    c = serving.PagedCache(k, k.clone(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), rope=(cos.cuda(), sin.cuda()))
    x = torch.randn(1, 7 * 64, generator=torch.Generator().manual_seed(0)).cuda()
    x[0, :64] = 0
    x[0, 64:128] *= 1e30
    x[0, 128:192] *= 1e-30
    x[0, 200] = float("inf")
    gain = torch.ones(64, device="cuda")
    ids = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    q = c.append(x, *ids, norm=(gain, gain), eps=1e-5)
    c.check()
    assert (q[0, :64] == 0).all()
    assert torch.allclose(q[0, 64:128].double().pow(2).mean(), torch.tensor(1.0, dtype=torch.float64, device="cuda"), rtol=1e-5)
    assert torch.isfinite(q[0, 128:192]).all() and (q[0, 128:192].abs() < 1e-24).all()
    assert not torch.isfinite(q[0, 192:256]).all() and torch.isfinite(q[0, 256:]).all()
    q = c.append(x, *ids, norm=(gain, None), eps=0.0)
    assert torch.isnan(q[0, :64]).all()
    assert torch.allclose(q[0, 128:192].double().pow(2).mean(), torch.tensor(1.0, dtype=torch.float64, device="cuda"), rtol=1e-5)


@pytest.mark.parametrize("act,size", [("f32", 2e38), ("bf16", 3e38), ("f32", 1e-40), ("bf16", 1e-39), ("f32", 1e-44)])
def test_ends_of_the_range(serving, act, size):
    """Heads whose factor leaves float32's normal numbers, without eps."""
    cos, sin = tables(4, 64)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device="cuda")
    c = serving.PagedCache(k, k.clone(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), rope=(cos.cuda(), sin.cuda()))
    x = ((torch.rand(1, 4 * 64, generator=torch.Generator().manual_seed(1)) * 1.0 + 0.1) / 1.1 * size).to(DT[act])
    gain = torch.ones(64, device="cuda")
    ids = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]   # position 0: no rotation
    q = c.append(x.cuda(), *ids, norm=(gain, gain), eps=0.0)
    c.check()
    xd = x.double()[:, :128].view(2, 64)
    want = (xd / xd.pow(2).mean(dim=1, keepdim=True).sqrt()).view(1, 128)
    # the factor and its product round to float32, then the result to its type
    tol = 2.01 * 2.0 ** -24 * want.abs()
    tol = tol + STEP[act] * (want.abs() + tol)
    assert ((q.cpu().double() - want).abs() <= tol).all()


def test_completing_form_graph_and_refusals(serving):
    import ctypes as C
    g = torch.Generator().manual_seed(4)
    cos, sin = (t.cuda() for t in tables(40, 64))
    k = torch.zeros(6, 2, 16, 64, dtype=torch.int8, device="cuda")
    scale = torch.full((2,), 0.05, device="cuda")
    table = torch.tensor([[0, 3], [4, 1]], dtype=torch.int32, device="cuda")
    c = serving.PagedCache(k, k.clone(), table, scale, scale, rope=(cos, sin))
    x = torch.randn(2, 8 * 64, generator=g).cuda()
    seq = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    pos = torch.tensor([30, 5], dtype=torch.int32, device="cuda")
    gains = [torch.randn(64, generator=g).cuda() for _ in range(2)]
    want = c.append(x, seq, pos, norm=gains)
    want_k = c.k.clone()
    c.k.zero_()
    out = torch.empty_like(want)
    rt = runtime()
    rt.call("tl_paged_append_norm", C.byref(c.desc), x, x.shape[1], 0, 2, 4, seq, pos, cos, sin, 40, gains[0], gains[1],
            C.c_double(1e-5), out, out.shape[1])
    assert torch.equal(out, want) and torch.equal(c.k, want_k)
    rt.close()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.append(x, seq, pos, norm=gains)
    for _ in range(3):
        x.copy_(torch.randn(2, 8 * 64, generator=g))
        pos.sub_(1)
        graph.replay()
        replayed = got.clone(), c.k.clone()
        assert torch.equal(c.append(x, seq, pos, norm=gains), replayed[0]) and torch.equal(c.k, replayed[1])
    c.check()
    for bad in ((gains[0].double(), None), (None, gains[0][:32]), (gains[0].cpu(), None), (gains[0].expand(1, 64), None),
                (torch.zeros(128, device="cuda")[::2], None), (torch.zeros(65, device="cuda")[1:], None), (gains[0],), (*gains, None)):
        with pytest.raises(ValueError):
            c.append(x, seq, pos, norm=bad)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            c.append(x, seq, pos, norm=gains, eps=eps)
