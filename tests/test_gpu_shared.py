"""Attention of rows that share the first positions of one sequence, against plain 64-bit attention."""
from __future__ import annotations

import math

import pytest

from gpu_util import runtime, torch as get_torch
from test_gpu_paged import DT, STEP, TINY, build, keys, make

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def reference(q, built, seq, pos, pseq, plen, page, scale, act, cache):
    """float64 attention of each row (keys 0 .. plen - 1 of pseq, plen .. pos of seq) and its error bound: that of
    attention_reference, n sums more for the prefix's parts, and probabilities of 16-bit rows in two 16-bit parts,
    each rounded to nearest, which keep 2^-17 (bfloat16) of them."""
    kv, hd = built[0][0].shape[1], built[0][0].shape[3]
    heads = q.shape[1] // hd
    want = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(want)
    qd = q.double().view(-1, heads, hd)
    pk, pv = (keys(built, w, pseq, plen, page) for w in (0, 1))
    own = {}
    for r in range(q.shape[0]):
        n = pos[r] + 1
        if seq[r] < 0 or n <= 0:
            continue
        k, v = pk[:n], pv[:n]
        if n > plen:
            if seq[r] not in own:
                most = max(p for s, p in zip(seq, pos) if s == seq[r]) + 1
                own[seq[r]] = own_keys(built, seq[r], plen, most, page)
            ko, vo = own[seq[r]]
            k, v = torch.cat([k, ko[:n - plen]]), torch.cat([v, vo[:n - plen]])
        for h in range(heads):
            kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            s = kh @ qd[r, h] * scale
            mag = (kh.abs() @ qd[r, h].abs()).max().item() * abs(scale)
            p = torch.softmax(s, 0)
            want[r, h] = p @ vh
            score = ((hd + 12) * 2.0 ** -24 + 2.0 ** -21) * mag * 1.4427 + 2.0 ** -22
            part = 2.0 ** -14 if cache == "bf16" and act == "bf16" else 2.0 ** -20
            tol[r, h] = (2 * score + part + 2 * (2 * n + 80) * 2.0 ** -24) * (p @ vh.abs())
    tol += STEP[act] * (want.abs() + tol) + TINY[act]
    return want.view(q.shape), tol.view(q.shape)


def own_keys(built, seq, first, end, page):
    """Positions first .. end - 1 of a sequence in float64, from its own pages."""
    out = []
    rows, table, _, scales, _ = built
    for which in (0, 1):
        pages = table[seq, first // page:-(-end // page)].long()
        x = rows[which][pages].transpose(1, 2).reshape(-1, rows[0].shape[1], rows[0].shape[3]).double()
        x = x[first % page:first % page + end - first]
        out.append(x if scales[which] is None else x * scales[which].double()[:, None])
    return out


def shared(cache, kv, hd, page, plen, lengths, seed=0, stride_pad=0):
    """Sequence 0 is the prompt; the others' table entries in front of their own first page are out of range, and
    what their page holds in front of it is NaN."""
    built = build(cache, kv, hd, page, [plen] + [plen + n for n in lengths], seed=seed, stride_pad=stride_pad)
    rows, table, wide, scales, g = built
    for i in range(1, len(lengths) + 1):
        if plen % page and cache != "i8" and plen // page < table.shape[1]:
            entry = int(table[i, plen // page])
            if 0 <= entry < rows[0].shape[0]:
                for r in rows:
                    r[entry, :, :plen % page] = float("nan")
        wide[i, :plen // page] = -1 if i % 2 else 2 ** 30
    return built


def check(got, want, tol):
    got = got.cpu().double()
    worst = ((got - want).abs() / tol.clamp_min(1e-300)).max().item()
    assert torch.isfinite(got).all() and worst <= 1, f"{worst} of the bound"


CASES = [
    # act, cache, query heads, KV heads, head dim, page, prefix, own keys of the rows' sequences
    ("f32", "i8", 8, 1, 64, 16, 1, [1, 3]),
    ("f32", "i8", 32, 4, 64, 8, 100, [1, 17, 64, 130]),
    ("f32", "i8", 32, 4, 64, 64, 500, [5] * 9),                  # more than 64 columns
    ("bf16", "i8", 5, 5, 128, 32, 33, [40, 77]),
    ("f16", "i8", 12, 1, 64, 1024, 700, [330, 12, 1]),
    ("f32", "i8", 16, 2, 128, 16, 257, [3, 1, 2, 9, 100, 31, 32, 33, 4]),
    ("f32", "f16", 6, 2, 128, 64, 64, [1, 63, 64, 300]),
    ("f16", "f16", 28, 4, 128, 16, 1000, [17, 260, 1]),
    ("f16", "f16", 28, 4, 128, 16, 999, [i % 7 + 1 for i in range(40)]),
    ("bf16", "f16", 8, 8, 64, 128, 300, [130, 5]),
    ("bf16", "f16", 8, 8, 64, 128, 127, [1 + i for i in range(70)]),
    ("f32", "bf16", 16, 2, 128, 16, 301, [1, 100, 301]),
    ("f32", "bf16", 16, 2, 128, 16, 75, [i % 5 + 1 for i in range(20)]),
    ("f32", "bf16", 3, 1, 64, 8, 9, [9, 200]),
    ("f16", "bf16", 4, 4, 64, 32, 66, [66, 31] * 40),
    ("bf16", "bf16", 40, 8, 128, 16, 2000, [15, 16, 200] * 9),
    ("bf16", "bf16", 32, 1, 64, 16, 45, [45]),
    ("f32", "i8", 4, 1, 64, 16, 9000, [1, 5000]),                 # split prefix, and an own part that is split and joined
    ("bf16", "bf16", 8, 1, 128, 64, 20011, [1, 2000, 3]),
    ("f32", "f16", 1, 1, 64, 8, 31, [1]), ("f32", "f16", 1, 1, 64, 8, 32, [1]), ("f32", "f16", 1, 1, 64, 8, 33, [96]),
]


@pytest.mark.parametrize("act,cache,heads,kv,hd,page,plen,own", CASES)
def test_shared(serving, act, cache, heads, kv, hd, page, plen, own):
    """Prefixes and own parts around tiles and pages; stale rows, unused pages and table entries hold NaN and numbers
    out of range; strides of their own; queued, in place and captured."""
    built = shared(cache, kv, hd, page, plen, own, seed=plen + heads, stride_pad=64)
    c = make(serving, built)
    g = built[4]
    b = len(own)
    wide = torch.randn(b, heads * hd + 16, generator=g).to(DT[act])
    q = wide.cuda()[:, :heads * hd]
    seq, pos = list(range(1, b + 1)), [plen + n - 1 for n in own]
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    out = torch.full((b, heads * hd + 8), 3.0, dtype=DT[act], device="cuda")
    c.attend_shared(q, *ids, 0, plen, out=out[:, :heads * hd])
    c.check()
    want, tol = reference(wide[:, :heads * hd], built, seq, pos, 0, plen, page, 1 / math.sqrt(hd), act, cache)
    check(out[:, :heads * hd], want, tol)
    assert (out[:, heads * hd:] == 3.0).all()
    again = q.clone()
    c.attend_shared(again, *ids, 0, plen, out=again)
    assert torch.equal(again, out[:, :heads * hd])
    graph = torch.cuda.CUDAGraph()
    captured = torch.empty_like(again)
    with torch.cuda.graph(graph):
        c.attend_shared(q, *ids, 0, plen, out=captured)
    for _ in range(3):
        captured.fill_(5.0)
        graph.replay()
        c.attend_shared(q, *ids, 0, plen, out=again)
        check(captured, want, tol)
    c.check()


@pytest.mark.parametrize("rows", [7, 90, 300])
@pytest.mark.parametrize("cache", ["i8", "bf16"])
def test_rows_of_every_kind(serving, rows, cache):
    """Rows before the prefix's end (they attend its keys up to their own, NaN behind them notwithstanding), at its end,
    behind it; rows without keys and padded ones; several rows of one sequence."""
    plen, page, kv, heads = 150, 16, 2, 8
    own = [1, 40, 300, 7]
    built = shared(cache, kv, 64, page, plen, own, seed=rows)
    g = built[4]
    seq, pos = [], []
    for i in range(rows):
        s = 1 + i % len(own)
        kind = i % 6
        seq.append(-1 if kind == 3 else s)
        pos.append(-1 if kind == 5 else plen - 1 if kind == 1 else (i * 31) % plen if kind == 2 else plen + (i * 17) % own[s - 1])
    c = make(serving, built)
    act = "f32" if cache == "i8" else "bf16"
    q = torch.randn(rows, heads * 64, generator=g).to(DT[act])
    want, tol = reference(q, built, seq, pos, 0, plen, page, 0.125, act, cache)
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    out = torch.full((rows, heads * 64), 5.0, dtype=DT[act], device="cuda")
    c.attend_shared(q.cuda(), *ids, 0, plen, out=out)
    c.check()
    live = [i for i in range(rows) if seq[i] >= 0]
    check(out[live], want[live], tol[live])
    assert (out[[i for i in range(rows) if seq[i] < 0]] == 5.0).all()
    # a prompt that is not written to its end: rows before it do not see what lies there
    if cache == "bf16":
        short = [i for i in live if pos[i] < 100]
        some = torch.tensor(short, device="cuda")
        for t in (c.k, c.v):
            for p in range(112 // page, -(-plen // page)):
                t[int(c.table[0, p])] = float("nan")
        got = c.attend_shared(q.cuda()[some].contiguous(), ids[0][some].contiguous(), ids[1][some].contiguous(), 0, plen)
        check(got, want[short], tol[short])


@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "bf16"), ("f32", "f16")])
def test_in_place_and_apart_are_the_same(serving, act, cache):
    """Rows shorter than the prefix, whose results may lie where the prefix's workgroups read q, change nothing in the
    other rows' last bits."""
    kv, hd, page, plen, b = 2, 64, 16, 3000, 60
    built = shared(cache, kv, hd, page, plen, [i % 40 + 1 for i in range(b)], seed=9)
    c = make(serving, built)
    seq = torch.arange(1, b + 1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([i * 7 % 90 if i % 2 else plen + i % 40 for i in range(b)], dtype=torch.int32, device="cuda")
    q = (3 * torch.randn(b, 8 * kv * hd, generator=built[4])).to(DT[act]).cuda()
    want = c.attend_shared(q, seq, pos, 0, plen)
    for _ in range(20):
        out = q.clone()
        c.attend_shared(out, seq, pos, 0, plen, out=out)
        assert torch.equal(out, want)
    c.check()


def test_equals_attend(serving):
    """Where the sequences' tables hold the prompt's pages, as a server's do, the result is attend's."""
    plen, page, kv, heads, b = 1000, 16, 2, 16, 24
    built = shared("f16", kv, 64, page, plen, [1 + 5 * i for i in range(b)], seed=1)
    c = make(serving, built)
    c.table[1:, :plen // page] = c.table[0, :plen // page]
    tail = plen % page
    for i in range(1, b + 1):   # the page that the prompt ends in is each sequence's own copy
        for t in (c.k, c.v):
            t[int(c.table[i, plen // page]), :, :tail] = t[int(c.table[0, plen // page]), :, :tail]
    q = torch.randn(b, heads * 64, generator=built[4]).cuda()
    seq = torch.arange(1, b + 1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([plen + 5 * i for i in range(b)], dtype=torch.int32, device="cuda")
    want = c.attend(q, seq, pos)
    for n in (1, 31, 500, plen):
        assert (c.attend_shared(q, seq, pos, 0, n) - want).abs().max() < 2e-6
    assert torch.equal(c.attend_shared(q, seq, pos, 0, 0), want)
    # a longer prefix than some rows' positions
    assert (c.attend_shared(q, seq, pos, b, plen + 5 * (b - 1) + 1)[b - 1] - want[b - 1]).abs().max() < 2e-6


def test_two_prompts_in_a_batch(serving):
    """One call for each prompt into one output, the other rows padded."""
    plen, page = 70, 16
    built = shared("f16", 1, 64, page, plen, [3, 4, 5, 6], seed=5)
    c = make(serving, built)
    q = torch.randn(4, 256, generator=built[4])
    pos = [plen + 2, plen + 3, plen + 4, plen + 5]
    out = torch.zeros(4, 256, device="cuda")
    dpos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    # sequence 4's own positions serve as the second prompt, as they lie in its table from 64 on
    first = torch.tensor([1, 2, -1, -1], dtype=torch.int32, device="cuda")
    second = torch.tensor([-1, -1, 3, 4], dtype=torch.int32, device="cuda")
    c.attend_shared(q.cuda(), first, dpos, 0, plen, out=out)
    assert (out[2:] == 0).all()
    c.attend_shared(q.cuda(), second, dpos, 0, plen, out=out)
    want, tol = reference(q, built, [1, 2, 3, 4], pos, 0, plen, page, 0.125, "f32", "f16")
    check(out, want, tol)


def test_scales_and_extreme_scores(serving):
    """A negative, a zero and a large scale; scores that differ by hundreds; alike keys."""
    plen, page = 300, 16
    built = shared("f16", 1, 64, page, plen, [9, 50], seed=7)
    c = make(serving, built)
    q = torch.randn(2, 8 * 64, generator=built[4])
    seq, pos = [1, 2], [plen + 8, plen + 49]
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    for scale in (-0.125, 0.0, 3.0, 1e-3, -5.0):
        got = c.attend_shared(q.cuda(), *ids, 0, plen, scale=scale)
        want, tol = reference(q, built, seq, pos, 0, plen, page, scale, "f32", "f16")
        check(got, want, tol)
    for big in (1e-20, 1e4, 1e20):   # rows whose parts need another power of two
        x = q * big
        got = c.attend_shared(x.cuda(), *ids, 0, plen, scale=0.125 / big)
        want, tol = reference(x, built, seq, pos, 0, plen, page, 0.125 / big, "f32", "f16")
        check(got, want, tol)


def test_faults_are_left_out(serving):
    """A page of the prefix out of range: its keys are left out and reported; every page so: NaN; own pages likewise."""
    plen, page = 64, 16
    built = shared("f16", 1, 64, page, plen, [1] * 10, seed=3)
    for lost in ([1], [0, 1, 2, 3]):
        c = make(serving, built)
        for p in lost:
            c.table[0, p] = 10 ** 6 if p % 2 else -1
        q = torch.randn(10, 8 * 64, generator=built[4])
        seq = torch.arange(1, 11, dtype=torch.int32, device="cuda")
        pos = torch.full((10,), plen, dtype=torch.int32, device="cuda")
        if lost != [1]:
            c.table[3, plen // page] = -5
        got = c.attend_shared(q.cuda(), seq, pos, 0, plen)
        with pytest.raises(ValueError, match="out of range"):
            c.check()
        c.check()
        kept = [t for t in range(plen) if t // page not in lost]
        pk, pv = (keys(built, w, 0, plen, page)[kept, 0] for w in (0, 1))
        for r in range(10):
            if lost != [1] and r == 2:
                assert torch.isnan(got[r]).all()
                continue
            ko, vo = own_keys(built, r + 1, plen, plen + 1, page)
            k, v = torch.cat([pk, ko[:, 0]]), torch.cat([pv, vo[:, 0]])
            want = torch.softmax(q[r].double().view(8, 64) @ k.t() / 8, 1) @ v
            assert (got[r].cpu().double().view(8, 64) - want).abs().max() < 1e-5
    c = make(serving, built)
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([1, 99, 2], [plen, plen, 10 ** 8])]
    out = torch.full((3, 512), 4.0, device="cuda")
    c.attend_shared(q[:3].cuda(), *ids, 0, plen, out=out)
    with pytest.raises(ValueError, match="out of range"):
        c.check()
    assert (out[1:] == 4.0).all() and not (out[0] == 4.0).any()


def test_many_rows(serving):
    """A block of a prompt's rows behind a shared prefix, and as many rows as fill several column blocks of each KV head."""
    plen, page, kv, heads = 333, 32, 2, 8
    built = shared("bf16", kv, 128, page, plen, [200, 3], seed=11)
    c = make(serving, built)
    rows = 201
    seq = [1] * 200 + [2]
    pos = [plen + i for i in range(200)] + [plen + 2]
    q = torch.randn(rows, heads * 128, generator=built[4]).to(torch.bfloat16)
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    got = c.attend_shared(q.cuda(), *ids, 0, plen)
    c.check()
    want, tol = reference(q, built, seq, pos, 0, plen, page, 1 / math.sqrt(128), "bf16", "bf16")
    check(got, want, tol)


def test_completing_form_streams_and_refusals(serving):
    import ctypes as C
    plen, page = 100, 16
    built = shared("i8", 2, 64, page, plen, [30, 1, 5], seed=2)
    c = make(serving, built)
    q = torch.randn(3, 8 * 64, generator=built[4]).cuda()
    seq = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    pos = torch.tensor([plen + 29, plen, plen + 4], dtype=torch.int32, device="cuda")
    want = c.attend_shared(q, seq, pos, 0, plen)
    rt = runtime()
    out = torch.empty_like(q)
    rt.call("tl_paged_attention_shared", C.byref(c.desc), q, 512, 0, 3, 8, seq, pos, 0, plen, C.c_float(0.125), out, 512)
    assert torch.equal(out, want)
    c.table[0, 2] = -1
    with pytest.raises(ValueError, match="out of range"):
        rt.call("tl_paged_attention_shared", C.byref(c.desc), q, 512, 0, 3, 8, seq, pos, 0, plen, C.c_float(0.125), out, 512)
    rt.close()
    c = make(serving, built)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append(c.attend_shared(q, seq, pos, 0, plen))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    for bad in ((0, -1), (0, c.table.shape[1] * page + 1), (4, 10), (-1, 10)):
        with pytest.raises(ValueError):
            c.attend_shared(q, seq, pos, *bad)
    with pytest.raises(ValueError):
        c.attend_shared(q.double(), seq, pos, 0, plen)
    with pytest.raises(ValueError):
        c.attend_shared(q[:, :448 + 32], seq, pos, 0, plen)
    assert c.attend_shared(q[:0], seq[:0], pos[:0], 0, plen).shape == (0, 512)
    c.check()


def test_offsets_past_32_bits(serving):
    """A prefix whose pages lie past 2^32 bytes into a cache."""
    page, kv, hd = 1024, 2, 64
    n_pages = 2 ** 32 // (page * kv * hd * 2) + 64
    k = torch.empty(n_pages, kv, page, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([[n_pages - 1, 0], [n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    for p in (n_pages - 1, 0, n_pages - 2):
        k[p].normal_()
        v[p].normal_()
    c = serving.PagedCache(k, v, table)
    q = torch.randn(1, 4 * hd, device="cuda", dtype=torch.float16)
    pos = torch.tensor([page + 500], dtype=torch.int32, device="cuda")
    got = c.attend_shared(q, torch.ones(1, dtype=torch.int32, device="cuda"), pos, 0, page + 100)
    c.check()
    kk, vv = (torch.cat([t[n_pages - 1, 1], t[0, 1, :100], t[n_pages - 2, 1, 100:501]]).double() for t in (k, v))
    for h in (2, 3):
        p = torch.softmax(kk @ q[0, h * hd:(h + 1) * hd].double() / 8, 0)
        assert (got[0, h * hd:(h + 1) * hd].double() - p @ vv).abs().max() < 2e-3
