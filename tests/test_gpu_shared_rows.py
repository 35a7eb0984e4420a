"""Attention over a shared prefix: what a row's result may depend on."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch
from test_gpu_paged import DT, make
from test_gpu_shared import shared

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def vector(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# others' q: numbers that move their maxima about, the largest, none at all
OTHERS = [lambda q, g: 9 * torch.randn(q.shape, generator=g), lambda q, g: torch.full(q.shape, 3e4),
          lambda q, g: torch.full(q.shape, float("nan")), lambda q, g: torch.full(q.shape, -float("inf")),
          lambda q, g: torch.zeros(q.shape)]
TYPES = [("f32", "i8"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "i8")]


@pytest.mark.parametrize("b", [12, 60])
@pytest.mark.parametrize("kind", ["live", "padded", "fault", "short"])
@pytest.mark.parametrize("act,cache", TYPES)
def test_a_row_is_its_own(serving, act, cache, kind, b):
    """A row's last bits are the same whatever the other rows of its batch ask for: live ones, padded ones and ones out of
    range whose positions lie behind the prefix, ones that end before it does."""
    kv, hd, page, plen = 2, 64, 16, 3000
    built = shared(cache, kv, hd, page, plen, [i % 40 + 1 for i in range(b)], seed=4)
    c = make(serving, built)
    g = built[4]
    pos = [plen + i % 40 for i in range(b)]
    seq = list(range(1, b + 1))
    other = [i for i in range(b) if i % 3 == 1]
    for i in other:
        if kind == "padded":
            seq[i] = -1
        elif kind == "fault":
            seq[i] = b + 5
        elif kind == "short":
            pos[i] = i * 7 % 90
    mine = [i for i in range(b) if i % 3 != 1]
    q = (5 * torch.randn(b, 4 * kv * hd, generator=g)).to(DT[act]).cuda()
    ids = vector(seq), vector(pos)
    want = c.attend_shared(q, *ids, 0, plen)[mine]
    assert torch.isfinite(want).all()
    for fill in OTHERS:
        q[other] = fill(q[other], g).to(DT[act]).cuda()
        assert torch.equal(c.attend_shared(q, *ids, 0, plen)[mine], want)
    if kind == "fault":
        with pytest.raises(ValueError, match="out of range"):
            c.check()
    c.check()


@pytest.mark.parametrize("act,cache", TYPES)
def test_two_prompts_in_place(serving, act, cache):
    """One call for each prompt with q's own rows as results: what the first call wrote over its rows, which pad the second
    call, changes nothing there."""
    kv, hd, page, plen, b = 2, 64, 16, 2000, 24
    built = shared(cache, kv, hd, page, plen, [plen + i for i in range(b)], seed=6)
    c = make(serving, built)
    # the second prompt: positions 0 .. of another sequence, which the first one's pages serve as well
    c.table[b, :plen // page] = c.table[0, :plen // page]
    q = (5 * torch.randn(b, 4 * kv * hd, generator=built[4])).to(DT[act]).cuda()
    pos = vector([2 * plen - 1 + i for i in range(b)])
    first = vector([i + 1 if i % 2 else -1 for i in range(b)])
    second = vector([-1 if i % 2 else i + 1 for i in range(b)])
    lens = plen, plen + 7
    want = torch.zeros_like(q)
    c.attend_shared(q, first, pos, 0, lens[0], out=want)
    c.attend_shared(q, second, pos, b, lens[1], out=want)
    x = q.clone()
    c.attend_shared(x, first, pos, 0, lens[0], out=x)
    c.attend_shared(x, second, pos, b, lens[1], out=x)
    c.check()
    assert torch.equal(x, want) and torch.isfinite(x).all()


@pytest.mark.parametrize("plen", [700, 704])
def test_prompts_by_slices(serving, plen):
    """Prompts whose rows stand together, one call each on slices of the batch's tensors, give what the padded calls give,
    but for the order in which sums are split.  The second prompt's own page holds NaN in front of position 700, which its
    rows attend: they are NaN, and no other row is."""
    kv, hd, page, b, cut = 2, 64, 16, 23, 5
    built = shared("f16", kv, hd, page, plen, [plen + i for i in range(b)], seed=8)
    c = make(serving, built)
    c.table[b, :plen // page] = c.table[0, :plen // page]
    wide = torch.randn(b, 4 * kv * hd + 16, generator=built[4]).cuda()
    q, pos = wide[:, :4 * kv * hd], vector([2 * plen - 1 + i for i in range(b)])
    seq = vector(list(range(1, b + 1)))
    prompts = [(slice(0, cut), 0, plen), (slice(cut, b), b, plen + 7)]
    want, got = torch.zeros(b, 4 * kv * hd, device="cuda"), torch.zeros(b, 4 * kv * hd, device="cuda")
    for rows, prefix, n in prompts:
        others = torch.full_like(seq, -1)
        others[rows] = seq[rows]
        c.attend_shared(q, others, pos, prefix, n, out=want)
        c.attend_shared(q[rows], seq[rows], pos[rows], prefix, n, out=got[rows])
    c.check()
    whole = b if plen % page == 0 else cut
    assert (got - want)[:whole].abs().max() < 2e-6 and (want[:whole] != 0).any(1).all()
    assert torch.isnan(got[whole:]).all() and torch.isnan(want[whole:]).all()
