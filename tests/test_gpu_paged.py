"""The paged KV cache: append with rotation, and the attention of one query row per
token, against plain 64-bit implementations."""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import dev, empty, host, runtime, torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
# a rounding is off by at most half a step: eps / 2
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# least normal numbers' half steps: what a subnormal rounding may lose
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def build(cache, kv, hd, page, lengths, seed=0, extra=2, stride_pad=0, stale=None, table_pad=1):
    """A pool and a table for sequences of the given lengths.  Pages are handed out in a
    shuffled order; unused pages, rows past a sequence's last and (16-bit) are filled
    with `stale`, table entries past the last with numbers out of range."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    n_pages = sum(need) + extra
    order = torch.randperm(n_pages, generator=g)
    cols = max(max(need, default=0), 1)
    table = torch.full((len(lengths), cols + table_pad), 2 ** 30, dtype=torch.int32)
    table[:, -1] = -7
    block = kv * page * hd
    pool = [torch.empty(n_pages, block + stride_pad, dtype=DT[cache]) for _ in range(2)]
    rows = []
    for p in pool:
        if cache == "i8":
            p.copy_(torch.randint(-127, 128, p.shape, generator=g))
        else:
            p.fill_(float("nan") if stale is None else stale)
        rows.append(p[:, :block].view(n_pages, kv, page, hd))
    at = 0
    for i, n in enumerate(lengths):
        table[i, :need[i]] = order[at: at + need[i]].to(torch.int32)
        at += need[i]
        if cache != "i8":
            for j in range(n):
                for r in rows:
                    r[table[i, j // page], :, j % page] = (torch.randn(kv, hd, generator=g) * 1.3).to(DT[cache])
    scales = [0.02 + 0.04 * torch.rand(kv, generator=g) for _ in range(2)] if cache == "i8" else [None, None]
    return rows, table[:, :cols], table, scales, g


def make(serving, built, rope=None):
    rows, _, wide, scales, _ = built
    cols = built[1].shape[1]
    # the views keep their page stride and the table its row stride on the device
    k, v = (torch.as_strided(r._base.cuda(), r.shape, r.stride()) for r in rows)
    table = wide.cuda()[:, :cols]
    return serving.PagedCache(k, v, table, *(None if s is None else s.cuda() for s in scales),
                              rope=None if rope is None else tuple(t.cuda() for t in rope))


def keys(built, which, seq, n, page):
    """The first n rows of a sequence in float64 [n][kv][hd]."""
    rows, table, _, scales, _ = built
    pages = table[seq, :-(-n // page)].long() if n else table[seq, :0].long()
    x = rows[which][pages].transpose(1, 2).reshape(-1, rows[0].shape[1], rows[0].shape[3])[:n].double()
    return x if scales[which] is None else x * scales[which].double()[:, None]


def attention_reference(q, built, seq, pos, page, scale, act, cache):
    """float64 attention of each row and its error bound (see below)."""
    kv, hd = built[0][0].shape[1], built[0][0].shape[3]
    heads = q.shape[1] // hd
    want = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(want)
    qd = q.double().view(-1, heads, hd)
    for r in range(q.shape[0]):
        n = pos[r] + 1
        if seq[r] < 0 or n <= 0:
            continue
        k, v = keys(built, 0, seq[r], n, page), keys(built, 1, seq[r], n, page)
        for h in range(heads):
            kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            s = kh @ qd[r, h] * scale
            mag = (kh.abs() @ qd[r, h].abs()).max().item() * abs(scale)
            p = torch.softmax(s, 0)
            want[r, h] = p @ vh
            # Score: hd products and sums (q's two 16-bit parts: within 2^-21 of it), the scale, the
            # base-2 conversion and the maximum's subtraction, each 2^-24 of a number of at most mag
            # log2(e); the exponential 2^-22.  A probability's parts keep 2^-20 of it (float16, or
            # three bfloat16 parts) or 2^-14 (two bfloat16 parts).  The sum over n keys, the wavefronts
            # and the splits adds (n + 40) 2^-24 of the sum of magnitudes; numerator and denominator.
            score = ((hd + 12) * 2.0 ** -24 + 2.0 ** -21) * mag * 1.4427 + 2.0 ** -22
            part = 2.0 ** -14 if cache == "bf16" and act == "bf16" else 2.0 ** -20
            tol[r, h] = (2 * score + part + 2 * (n + 40) * 2.0 ** -24) * (p @ vh.abs())
    tol += STEP[act] * (want.abs() + tol) + TINY[act]
    return want.view(q.shape), tol.view(q.shape)


CASES = [
    # act, cache, query heads, KV heads, head dim, page, positions of the rows (-1: no keys)
    ("f32", "i8", 8, 1, 64, 16, [0, 1, 6, 7, 8, 15, 16, 31, 32, 33, 63, 127, 128, -1]),
    ("f32", "i8", 32, 4, 64, 8, [500, 3, 129, 255, 256]),
    ("bf16", "i8", 5, 5, 128, 32, [40, 77, -1]),
    ("f16", "i8", 12, 1, 64, 1024, [1029, 12]),               # more than 8 query heads of a KV head
    ("f32", "f16", 6, 2, 128, 64, [0, 63, 64, 300]),
    ("f16", "f16", 28, 4, 128, 16, [17, 1000, 260]),
    ("bf16", "f16", 8, 8, 64, 128, [130, 5]),
    ("f32", "bf16", 16, 2, 128, 16, [0, 100, 301]),           # third parts
    ("f32", "bf16", 3, 1, 64, 8, [9, 200]),
    ("f16", "bf16", 4, 4, 64, 32, [66, 31]),
    ("bf16", "bf16", 40, 8, 128, 16, [15, 16, 200]),
    ("bf16", "bf16", 32, 1, 64, 16, [45]),                    # four blocks of 8 query heads
    ("f32", "i8", 4, 1, 64, 16, [9000]),                      # split over workgroups and joined
    ("bf16", "bf16", 8, 1, 128, 64, [20011]),
]


@pytest.mark.parametrize("act,cache,heads,kv,hd,page,positions", CASES)
def test_attention(serving, act, cache, heads, kv, hd, page, positions):
    """Lengths of zero, one, around tiles and pages; stale rows, unused pages and table entries hold
    NaN and numbers out of range; rows and pages with strides of their own."""
    built = build(cache, kv, hd, page, [p + 1 for p in positions], seed=len(positions) + heads, stride_pad=64)
    c = make(serving, built)
    g = built[4]
    b = len(positions)
    wide = (torch.randn(b, heads * hd + 16, generator=g)).to(DT[act])
    q = wide.cuda()[:, :heads * hd]
    out = torch.full((b, heads * hd + 8), 3.0, dtype=DT[act], device="cuda")
    c.attend(q, None, torch.tensor(positions, dtype=torch.int32, device="cuda"), out=out[:, :heads * hd])
    c.check()
    want, tol = attention_reference(wide[:, :heads * hd], built, list(range(b)), positions, page, 1 / math.sqrt(hd), act, cache)
    got = out[:, :heads * hd].cpu().double()
    worst = ((got - want).abs() / tol.clamp_min(1e-300)).max().item()
    assert torch.isfinite(got).all() and worst <= 1, f"{worst} of the bound"
    assert (out[:, heads * hd:] == 3.0).all()
    for i, p in enumerate(positions):
        if p < 0:
            assert (got[i] == 0).all()


@pytest.mark.parametrize("rows,longest,cache,kv,heads", [
    (65, 700, "i8", 2, 8), (130, 300, "f16", 1, 16), (257, 260, "i8", 1, 9), (600, 150, "bf16", 2, 4),
    (20, 12000, "f16", 1, 8)])       # the last: one row of 94 parts among short ones
def test_attention_many_rows(serving, rows, longest, cache, kv, heads):
    """Rows past one lane each and past one workgroup's threads, padded ones and ones without keys among them; parts
    joined in place and, captured, by a kernel of their own."""
    seqs = min(rows, 24)
    lengths = [longest if i == seqs // 2 else 1 + (i * 37) % min(longest, 140) for i in range(seqs)]
    built = build(cache, kv, 64, 16, lengths, seed=rows, stale=0.0)
    c = make(serving, built)
    g = built[4]
    seq = [i % seqs if i % 11 != 3 else -1 for i in range(rows)]
    pos = [-1 if i % 13 == 5 else lengths[s] - 1 - (i // seqs) % lengths[s] for i, s in enumerate(seq)]
    q = torch.randn(rows, heads * 64, generator=g)
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    want, tol = attention_reference(q, built, seq, pos, 16, 0.125, "f32", cache)
    qd = q.cuda()
    out = torch.full((rows, heads * 64), 5.0, device="cuda")
    c.attend(qd, *ids, out=out)
    graph = torch.cuda.CUDAGraph()
    captured = torch.full((rows, heads * 64), 5.0, device="cuda")
    with torch.cuda.graph(graph):
        c.attend(qd, *ids, out=captured)
    for _ in range(3):
        graph.replay()
        c.attend(qd, *ids, out=out)
        c.check()
        for o in (out, captured):
            got = o.cpu().double()
            for r in range(rows):
                if seq[r] < 0:
                    assert (got[r] == 5.0).all()
                    got[r] = 0
            assert torch.isfinite(got).all() and ((got - want).abs() <= tol + 1e-300).all()


def test_attention_completing_form_and_causal_rows(serving):
    """tl_paged_attention (the handle's stream and scratch) gives the same bits; several rows of one sequence
    at rising positions are causal attention; padded rows stay as they were."""
    import ctypes as C
    built = build("i8", 2, 64, 16, [70, 3000], seed=3)
    c = make(serving, built)
    seq, pos = [0, 1, -1, 0, 0, 1, -5], [69, 2999, 10, 68, 67, 0, 5]
    q = torch.randn(7, 8 * 64, generator=built[4])
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    out = torch.full((7, 512), 7.5, device="cuda")
    c.attend(q.cuda(), *ids, scale=0.3, out=out)
    rt = runtime()
    again = torch.full((7, 512), 7.5, device="cuda")
    for _ in range(2):
        rt.call("tl_paged_attention", C.byref(c.desc), q.cuda(), 512, 0, 7, 8, *ids, 0.3, again, 512)
    assert torch.equal(out, again)
    want, tol = attention_reference(q, built, seq, pos, 16, 0.3, "f32", "i8")
    got = out.cpu().double()
    for r in (2, 6):
        assert (got[r] == 7.5).all()
        got[r] = 0
    assert ((got - want).abs() <= tol + 1e-300).all()
    rt.close()


def test_attention_faults_are_left_out(serving):
    """Keys of a page out of range take no part; a sequence or position out of range leaves its row alone.
    Both are reported, by either form."""
    import ctypes as C
    built = build("f16", 1, 64, 16, [100, 40], seed=5, table_pad=0)
    rows, table, wide, _, g = built
    c = make(serving, built)
    q = torch.randn(4, 128, generator=g)
    good = c.table.clone()
    c.table[0, 2] = -3
    c.table[0, 4] = 10 ** 6
    pos = torch.tensor([99, 39, 5, 7 * 16], dtype=torch.int32, device="cuda")     # the last: past the table
    seq = torch.tensor([0, 1, 2, 1], dtype=torch.int32, device="cuda")            # the third: no such sequence
    out = torch.full((4, 128), 9.0, device="cuda")
    c.attend(q.cuda(), seq, pos, out=out)
    with pytest.raises(ValueError, match="out of range"):
        c.check()
    c.check()
    left = [t for t in range(100) if not 32 <= t < 48 and not 64 <= t < 80]
    k, v = (keys(built, w, 0, 100, 16)[left, 0] for w in (0, 1))
    for h in range(2):
        p = torch.softmax(k @ q[0].double().view(2, 64)[h] / 8, 0)
        assert (out[0].cpu().double().view(2, 64)[h] - p @ v).abs().max() < 1e-5
    assert torch.isfinite(out[1]).all() and (out[2:] == 9.0).all()
    rt = runtime()
    with pytest.raises(ValueError, match="out of range"):
        rt.call("tl_paged_attention", C.byref(c.desc), q.cuda(), 128, 0, 4, 2, seq, pos, 0.125, out, 128)
    c.table.copy_(good)
    rt.call("tl_paged_attention", C.byref(c.desc), q.cuda(), 128, 0, 2, 2, seq, pos, 0.125, out, 128)
    # every page of a row out of range: no keys at all, as a softmax over none is: not a number
    c.table[1] = -1
    c.attend(q[:1].cuda(), torch.tensor([1], dtype=torch.int32, device="cuda"), pos[1:2], out=out[:1])
    assert torch.isnan(out[0]).all()
    rt.close()


def test_attention_in_place_and_scales(serving):
    """out = q gives the bits of another out, whole rows and split ones; scales of zero and below."""
    built = build("f16", 2, 64, 16, [5000, 90, 300], seed=6)
    c = make(serving, built)
    q = torch.randn(3, 24 * 64, generator=built[4])
    pos = torch.tensor([4999, 89, -1], dtype=torch.int32, device="cuda")
    for scale in (0.125, 0.0, -0.2):
        x = q.cuda()
        out = c.attend(x, None, pos, scale=scale)
        want, tol = attention_reference(q, built, [0, 1, 2], [4999, 89, -1], 16, scale, "f32", "f16")
        assert ((out.cpu().double() - want).abs() <= tol + 1e-300).all()
        assert c.attend(x, None, pos, scale=scale, out=x) is x and torch.equal(x, out)
    wide = torch.randn(3, 2 * 24 * 64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        c.attend(wide[:, :24 * 64], None, pos, out=wide[:, 64:25 * 64])
    c.attend(wide[:, :24 * 64], None, pos, out=wide[:, 24 * 64:])


def test_attention_extreme_scores(serving):
    """Scores far apart (all weight on one key), equal scores (plain means), a zero query, tiny and huge
    queries, and attended infinities and NaN."""
    built = build("f16", 1, 64, 16, [300], seed=8, stale=0.0)
    c = make(serving, built)
    v = keys(built, 1, 0, 300, 16)[:, 0]
    k = keys(built, 0, 0, 300, 16)[:, 0]
    pos = torch.full((5,), 299, dtype=torch.int32, device="cuda")
    seq = torch.zeros(5, dtype=torch.int32, device="cuda")
    q = torch.randn(5, 64, generator=built[4])
    q[0] *= 1e6
    q[1] = 0
    q[2] *= 1e-30
    q[3] *= 1e30
    got = c.attend(q.cuda(), seq, pos).cpu().double()
    for r in (0, 3):
        top = (k @ q[r].double()).argmax()
        assert (got[r] - v[top]).abs().max() <= 2.0 ** -20 * v[top].abs().max()
    for r in (1, 2):
        assert (got[r] - v.mean(0)).abs().max() <= 400 * 2.0 ** -24 * v.abs().mean(0).max() * 2
    q[4, 3] = float("inf")
    q[3, 0] = float("nan")
    got = c.attend(q.cuda(), seq, pos)
    assert torch.isnan(got[3:]).all() and torch.isfinite(got[:3]).all()
    c.v[c.table[0, 1].long(), 0, 3, 5] = float("nan")
    c.v[c.table[0, 1].long(), 0, 3, 6] = float("inf")
    got = c.attend(q[:3].cuda(), seq[:3], pos[:3])
    assert torch.isnan(got[1:, 5]).all() and not torch.isfinite(got[1:, 6]).any()
    rest = [d for d in range(64) if d not in (5, 6)]
    assert torch.isfinite(got[:, rest]).all()
    # the stale position after the last is not read: a shorter row does not see it
    got = c.attend(q[:3].cuda(), seq[:3], torch.full((3,), 18, dtype=torch.int32, device="cuda"))
    assert torch.isfinite(got).all()


def append_reference(qkv, seq, pos, cos, sin, heads, kv, hd):
    """float64 rotation of q and k, and v."""
    x = qkv.double().view(-1, heads + 2 * kv, hd)
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    turned = torch.cat([-qk[..., hd // 2:], qk[..., :hd // 2]], -1)
    p = torch.tensor(pos)
    c, s = cos.double()[p][:, None], sin.double()[p][:, None]
    # two products and their sum in float32
    tol = 3 * 2.0 ** -24 * ((qk * c).abs() + (turned * s).abs())
    return qk * c + turned * s, v, tol


def rope(n, hd):
    from lpta import build_rope_cache
    return tuple(torch.from_numpy(t) for t in build_rope_cache(n, hd, 10000.0))


@pytest.mark.parametrize("act,cache,heads,kv,hd,page", [
    ("f32", "i8", 32, 4, 64, 16), ("f32", "f16", 3, 1, 128, 8), ("f32", "bf16", 8, 8, 64, 64), ("bf16", "bf16", 32, 8, 128, 16),
    ("f16", "f16", 28, 4, 128, 1024), ("bf16", "i8", 5, 1, 64, 32), ("f16", "i8", 4, 4, 128, 16), ("bf16", "f16", 0, 2, 64, 16),
])
def test_append(serving, act, cache, heads, kv, hd, page):
    """One row of many sequences and many rows of one, odd positions, padded rows; only the named places
    change, and INT8 rows are the float32 steps' bits."""
    n_pos = 2 * page + 37
    lengths = [n_pos, 1, page + 1, n_pos - 3]
    built = build(cache, kv, hd, page, lengths, seed=heads + hd, stride_pad=32, stale=5.0)
    cos, sin = rope(n_pos, hd)
    c = make(serving, built, (cos, sin))
    seq = [0] * (n_pos - 5) + [1, -1, 2, 3, -2, 3]
    pos = list(range(n_pos - 5)) + [0, 3, page, n_pos - 4, -9, 1]
    rows, width = len(seq), (heads + 2 * kv) * hd
    wide = (torch.randn(rows, width + 24, generator=built[4]) * 2).to(DT[act])
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    before = [t.clone() for t in (c.k, c.v)]
    out = torch.full((rows, heads * hd + 8), 4.0, dtype=DT[act], device="cuda")
    c.append(wide.cuda()[:, :width], *ids, out=out[:, :heads * hd])
    c.check()
    use = [r for r in range(rows) if seq[r] >= 0]
    qk, v, tol = append_reference(wide[use][:, :width], None, [pos[r] for r in use], cos, sin, heads, kv, hd)
    got = out.cpu().double()
    assert (got[:, heads * hd:] == 4.0).all()
    assert all((got[r] == 4.0).all() for r in range(rows) if seq[r] < 0)
    err = (got[use][:, :heads * hd].view(len(use), heads, hd) - qk[:, :heads]).abs()
    assert (err <= tol[:, :heads] + STEP[act] * (qk[:, :heads].abs() + tol[:, :heads]) + TINY[act]).all()
    table = built[1]
    f32 = wide[use][:, :width].float().view(-1, heads + 2 * kv, hd).numpy()
    for which, (t, was) in enumerate(zip((c.k, c.v), before)):
        t, was = t.cpu(), was.cpu()
        places = torch.zeros(t.shape[0], t.shape[2], dtype=torch.bool)
        for i, r in enumerate(use):
            page_of, at = int(table[seq[r], pos[r] // page]), pos[r] % page
            places[page_of, at] = True
            row = t[page_of, :, at]
            x = qk[i, heads:] if which == 0 else v[i]
            if cache == "i8":
                y = f32[i, heads + kv:]
                if which == 0:
                    a = f32[i, heads:heads + kv]
                    turned = np.concatenate([-a[:, hd // 2:], a[:, :hd // 2]], 1)
                    y = a * cos[pos[r]].numpy() + turned * sin[pos[r]].numpy()
                y = np.clip(np.rint(y / built[3][which].numpy()[:, None]), -127, 127).astype(np.int8)
                assert np.array_equal(row.numpy(), y), (which, r)
            else:
                tl = tol[i, heads:] if which == 0 else torch.zeros_like(x)
                assert ((row.double() - x).abs() <= tl + STEP[cache] * (x.abs() + tl) + TINY[cache]).all(), (which, r)
        same = (t == was).all(dim=(1))
        assert same.all(dim=-1)[~places].all()


def test_append_equals_dense_cache(serving):
    """INT8 rows of 64-wide heads are bit for bit what tl_qkv_append writes into the dense cache, and q its
    rotated query."""
    rt = runtime()
    cfg = rt.cfg
    rows, heads, kv, hd = 37, cfg["n_heads"], cfg["n_kv_heads"], 64
    rng = np.random.default_rng(4)
    qkv = (rng.standard_normal((rows, (heads + 2 * kv) * hd)) * 2).astype(np.float32)
    sk, sv = (rng.uniform(0.02, 0.06, (1, kv)).astype(np.float32) for _ in range(2))
    cos, sin = rope(cfg["max_pos"], hd)
    rt.call("tl_set_kv_scales", sk, sv)
    rt.call("tl_set_rope_table", cos.numpy(), sin.numpy(), cfg["max_pos"])
    q8, qs, q_rot = empty((rows, heads * hd), np.int8), empty((rows,), np.float64), empty((rows, heads * hd), np.float32)
    rt.call("tl_qkv_append", 0, 0, 100, rows, dev(qkv), q8, qs, q_rot)
    table = torch.tensor([[8, 3, 5, 1, 9, 2, 0, 7, 6]], dtype=torch.int32, device="cuda")
    k = torch.zeros(10, kv, 16, hd, dtype=torch.int8, device="cuda")
    c = serving.PagedCache(k, torch.zeros_like(k), table, dev(sk[0]), dev(sv[0]), rope=(cos.cuda(), sin.cuda()))
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.arange(100, 100 + rows, dtype=torch.int32, device="cuda")
    q = c.append(dev(qkv), *ids)
    assert np.array_equal(host(q).view(np.uint32), host(q_rot).view(np.uint32))
    for g in range(kv):
        dk, dv = np.empty((rows, hd), np.int8), np.empty((rows, hd), np.int8)
        rt.call("tl_kv_read", 0, 0, g, 100, rows, dk, dv)
        for t, want in ((c.k, dk), (c.v, dv)):
            flat = host(t[table[0].long(), g].reshape(-1, hd))[100:100 + rows]
            assert np.array_equal(flat, want)
    # the completing form, in place
    import ctypes as C
    x = dev(qkv)
    c.k.zero_()
    rt.call("tl_paged_append", C.byref(c.desc), x, x.shape[1], 0, rows, heads, *ids, cos.cuda(), sin.cuda(), cos.shape[0],
            x, x.shape[1])
    assert torch.equal(x[:, :heads * hd], q)
    flat = host(c.k[table[0].long(), kv - 1].reshape(-1, hd))[100:100 + rows]
    rt.call("tl_kv_read", 0, 0, kv - 1, 100, rows, dk, dv)
    assert np.array_equal(flat, dk)
    rt.close()


def test_append_faults(serving):
    """A sequence, position, rotation row or page out of range: the row is skipped and reported."""
    built = build("f16", 2, 64, 16, [64, 64], seed=1, stale=1.0)
    c = make(serving, built, rope(60, 64))
    c.table[1, 1] = 99
    before = c.k.clone()
    seq, pos = [0, 5, 0, 0, 1, 0], [-1, 0, 60, 64, 20, 3]
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    q = torch.full((6, 64), 2.0, dtype=torch.float16, device="cuda")
    qkv = torch.randn(6, 5 * 64, generator=built[4]).to(torch.float16).cuda()
    c.append(qkv, *ids, out=q)
    with pytest.raises(ValueError, match="out of range"):
        c.check()
    assert (q[:5] == 2.0).all() and not (q[5] == 2.0).all()
    changed = (c.k != before).any(dim=3).any(dim=1).nonzero().tolist()
    assert changed == [[int(c.table[0, 0]), 3]]


def test_refusals(serving):
    built = build("bf16", 2, 64, 16, [20], seed=1)
    c = make(serving, built, rope(32, 64))
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: c.attend(q.double(), None, z), lambda: c.attend(q.cpu(), None, z), lambda: c.attend(q[:, :100], None, z),
                lambda: c.attend(q[:, :192], None, z), lambda: c.attend(q, None, z.long()), lambda: c.attend(q, None, z.cpu()),
                lambda: c.attend(q, None, torch.cat([z, z])), lambda: c.attend(q, torch.cat([z, z]), z),
                lambda: c.attend(q, None, z, out=q.float()), lambda: c.attend(q, None, z, out=q[:, :128]),
                lambda: c.attend(q[0], None, z), lambda: c.attend(q.t().contiguous().t().expand(1, 256)[:, ::2], None, z),
                lambda: c.append(q[:, :192], None, z), lambda: c.append(q[:, :100], None, z),
                lambda: make(serving, built).append(q, None, z),
                lambda: c.attend(torch.zeros(3, 260, dtype=torch.bfloat16, device="cuda")[:, 1:257], None, torch.cat([z, z, z])),
                lambda: serving.PagedCache(c.k.float(), c.v.float(), c.table), lambda: serving.PagedCache(c.k, c.v[:1], c.table),
                lambda: serving.PagedCache(c.k, c.v, c.table.long()), lambda: serving.PagedCache(c.k, c.v, c.table, z.float(), z.float()),
                lambda: serving.PagedCache(c.k.transpose(1, 2), c.v.transpose(1, 2), c.table),
                lambda: serving.PagedCache(c.k[..., :32], c.v[..., :32], c.table),
                lambda: serving.PagedCache(c.k.to(torch.int8), c.v.to(torch.int8), c.table),
                lambda: serving.PagedCache(c.k, c.v, c.table, rope=rope(10, 64))):
        with pytest.raises(ValueError):
            bad()
    assert c.attend(q[:0], None, z[:0]).shape == (0, 256) and c.append(q[:0], None, z[:0]).shape == (0, 0)


def test_graphs_and_streams(serving):
    """append + attend captured: replays follow the buffers, two graphs with scratch of their own replay side by side
    on two streams, and calls on a side stream use that stream."""
    built = build("i8", 2, 64, 16, [3000, 2000], seed=9)
    c = make(serving, built, rope(3100, 64))
    g = built[4]
    graphs = []
    side = torch.cuda.Stream()
    for n in range(2):
        qkv = torch.randn(1, 12 * 64, generator=g).cuda()
        seq = torch.tensor([n], dtype=torch.int32, device="cuda")
        pos = torch.tensor([1500 + n], dtype=torch.int32, device="cuda")
        with torch.cuda.stream(side):   # warm
            c.attend(c.append(qkv, seq, pos), seq, pos)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.attend(c.append(qkv, seq, pos), seq, pos)
        graphs.append((graph, qkv, seq, pos, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(6):
        for graph, qkv, seq, pos, out in graphs:
            qkv.copy_(torch.randn(1, 12 * 64, generator=g))
            pos.add_(37)
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, qkv, seq, pos, out in graphs:
            with torch.cuda.stream(side):
                want = c.attend(c.append(qkv, seq, pos), seq, pos)
            side.synchronize()
            assert torch.equal(out, want), step
    c.check()


def test_offsets_past_32_bits(serving):
    """A cache of more than 2^32 bytes: pages at its far end are written and read."""
    page, kv, hd = 1024, 2, 64
    n_pages = 2 ** 32 // (page * kv * hd * 2) + 64
    k = torch.empty(n_pages, kv, page, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device="cuda")
    c = serving.PagedCache(k, v, table, rope=tuple(t.cuda() for t in rope(3 * page, hd)))
    for p in table[0].tolist():
        k[p].normal_()
        v[p].normal_()
    ids = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([2 * page + 5], dtype=torch.int32, device="cuda")
    qkv = torch.randn(1, 6 * hd, device="cuda", dtype=torch.float16)
    q = c.append(qkv, *ids)
    assert torch.equal(v[n_pages - 2, :, 5].reshape(-1), qkv[0, 4 * hd:])
    out = c.attend(q, *ids)
    c.check()
    pages = table[0].long()
    n = 2 * page + 6
    kk, vv = (t[pages].transpose(1, 2).reshape(-1, kv, hd)[:n, :1].double()[:, 0] for t in (k, v))
    p = torch.softmax(kk @ q[0, :hd].double() / 8, 0)
    assert (out[0, :hd].double() - p @ vv).abs().max() < 2e-3
