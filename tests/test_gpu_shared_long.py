"""Attention over shared prefixes as long as take the launch's other forms, against 64 bits."""
from __future__ import annotations

import math

import pytest

from gpu_util import torch as get_torch
from test_gpu_paged import DT, STEP, TINY

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def vector(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("act,cache,heads,kv,hd,page,rows,plen,least", [
    # workgroups of both kinds take turns, 256 at a time: three column blocks, a number of them that 8 does not divide
    ("f32", "i8", 8, 1, 64, 16, 40, 22100, 256),
    ("bf16", "bf16", 8, 1, 128, 64, 40, 22100, 256),
    # two workgroups to a CU: four column blocks of each of three KV heads
    ("f16", "f16", 24, 3, 64, 64, 64, 87400, 512),
])
def test_long_prefixes(serving, act, cache, heads, kv, hd, page, rows, plen, least):
    """Prefixes that fill the GPU, beside as many workgroups of the rows' own keys, against 64 bits."""
    g = torch.Generator("cuda").manual_seed(plen + hd)
    own = [1 + i * 7 % 60 for i in range(rows)]
    first = -(-plen // page)
    counts = [first] + [-(-(plen + n) // page) - plen // page for n in own]
    n_pages = sum(counts) + 3
    pool = [torch.empty(n_pages, kv, page, hd, dtype=DT[cache], device="cuda") for _ in range(2)]
    for t in pool:
        x = torch.randn(t.shape, generator=g, device="cuda")
        t.copy_((x * 40).round().clamp(-127, 127) if cache == "i8" else x)
    scales = [torch.rand(kv, generator=g, device="cuda") * 0.01 + 0.02 for _ in range(2)] if cache == "i8" else [None, None]
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((1 + rows, plen // page + max(counts[1:])), -1, dtype=torch.int32, device="cuda")
    table[0, :first] = order[:first]
    at = first
    for i, n in enumerate(counts[1:], 1):
        table[i, plen // page:plen // page + n] = order[at:at + n]
        at += n
    c = serving.PagedCache(*pool, table, *scales)

    # how the call is split, from its scratch: the own keys' workgroups, then the prefix's splits
    part = c._scratch_bytes(rows, heads)
    workgroups = part // (2 * 8 * (hd + 2) * 4)
    more = (c._scratch_bytes(rows, heads, plen) - (part + 15) // 16 * 16) // 4 - rows - 1
    splits = more // (rows * heads * (hd + 2)) - 1
    grid = -(-rows * (heads // kv) // 128) * kv * splits
    assert workgroups >= least // 2 and workgroups >= 256 and grid >= least and grid % 8

    q = (1.5 * torch.randn(rows, heads * hd, generator=g, device="cuda")).to(DT[act])
    ids = vector(list(range(1, rows + 1))), vector([plen + n - 1 for n in own])
    got = c.attend_shared(q, *ids, 0, plen)
    for _ in range(2):
        assert torch.equal(c.attend_shared(q, *ids, 0, plen), got)
    c.check()

    def rows_of(which, pages, lo, n, h):
        x = pool[which][pages.long(), h].reshape(-1, hd)[lo:lo + n].double()
        return x if scales[which] is None else x * scales[which][h].double()
    for r in sorted({0, 1, rows // 2, rows - 2, rows - 1}):
        for h in range(kv):
            k, v = (torch.cat([rows_of(w, table[0, :first], 0, plen, h),
                               rows_of(w, table[r + 1, plen // page:plen // page + counts[r + 1]], plen % page, own[r], h)])
                    for w in (0, 1))
            rep = heads // kv
            qh = q[r].view(heads, hd)[h * rep:(h + 1) * rep].double()
            p = torch.softmax(qh @ k.t() / math.sqrt(hd), 1)
            want = p @ v
            # The bound of the shorter prefixes' test, but for the sums: an element passes through as many as its split has
            # keys, or the row's own, a tile's more, and one for each part that is joined; as much in the divisor
            mag = ((qh.abs() @ k.abs().t()).amax(1) / math.sqrt(hd))[:, None]
            score = ((hd + 12) * 2.0 ** -24 + 2.0 ** -21) * mag * 1.4427 + 2.0 ** -22
            part = 2.0 ** -14 if cache == "bf16" and act == "bf16" else 2.0 ** -20
            sums = -(-plen // splits) + own[r] + 64 + splits + 80
            tol = (2 * score + part + 2 * 2 * sums * 2.0 ** -24) * (p @ v.abs())
            tol = tol + STEP[act] * (want.abs() + tol) + TINY[act]
            off = (got[r].view(heads, hd)[h * rep:(h + 1) * rep].double() - want).abs()
            worst = (off / tol).max().item()
            assert worst <= 1, f"row {r}, KV head {h}: {worst} of the bound"
