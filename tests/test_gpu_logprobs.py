"""Log probabilities of given tokens, entropy and top alternatives against 64-bit NumPy, and Engine.score_tokens."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import runtime, torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Terms of the sums are off by 2^-23 (the exponential) and 3 2^-24 |y| of themselves (the difference to the
# maximum, its conversion to base 2), sums by 2^-24 for each of at most 60 additions on a term's way; |y|
# weighs in by its probability, less than 25 in all below.  So S is within EPS of itself.
EPS = 200 * 2.0 ** -24


@pytest.fixture(scope="module")
def serving():
    from lpta import serving
    return serving


def reference(x, targets, top):
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        ls = np.log(np.exp(x - m).sum(1, keepdims=True))
        lp = x - m - ls
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * lp, 0).sum(1)
    ids = np.stack([np.lexsort((np.arange(x.shape[1]), -r))[:top] for r in x]) if top else np.zeros((len(x), 0), int)
    picked = np.array([0.0 if t < 0 else lp[r, t] for r, t in enumerate(targets)])
    return picked, entropy, ids, np.take_along_axis(lp, ids, 1)


def check(got, x, targets, top, rows=None):
    lp, entropy, ids, tops = reference(x, targets, top)
    g = [t.cpu().numpy() for t in got]
    rows = np.arange(len(x)) if rows is None else rows
    # x - m rounds once, the difference once more
    with np.errstate(invalid="ignore"):
        off = lambda v: EPS + 2.0 ** -22 * (np.abs(v) + 25)   # noqa: E731
        assert (np.abs(g[0] - lp) <= off(lp))[rows][lp[rows] > -np.inf].all()
        assert (np.abs(g[1] - entropy) <= EPS * (1 + 3 * entropy))[rows].all()
        assert np.array_equal(g[2][rows], ids[rows])
        fine = np.isfinite(tops[rows])
        assert (np.abs(g[3] - tops) <= off(tops))[rows][fine].all()
        assert np.array_equal(g[3][rows][~fine], tops[rows][~fine])
    assert ((g[0] == -np.inf) == (lp == -np.inf))[rows].all()


@pytest.mark.parametrize("dtype,rows,vocab,top", [
    ("f32", 3, 1, 1), ("f32", 2, 7, 3), ("bf16", 3, 33, 32), ("f32", 4, 1000, 5), ("f16", 5, 2049, 32),
    ("f32", 2, 8184, 20), ("bf16", 9, 8185, 20), ("f16", 3, 8192, 1), ("f32", 5, 8193, 32), ("bf16", 17, 16385, 7),
    ("f32", 3, 32000, 0), ("f32", 40, 32000, 20), ("bf16", 11, 100003, 32), ("f16", 2, 300007, 10), ("f32", 1, 1200001, 32),
])
def test_logprobs(serving, dtype, rows, vocab, top):
    """Vocabularies around the parts' sizes, odd ones (rows at every alignment), strided rows, many equal logits in
    the 16-bit types."""
    rng = np.random.default_rng(vocab + rows)
    wide = (rng.standard_normal((rows, vocab + 5)) * 3).astype(np.float32)
    wide[:, :vocab:97] += 4
    t = torch.from_numpy(wide).to(DT[dtype])
    x = t[:, :vocab].float().numpy()
    targets = rng.integers(-1, vocab, rows).astype(np.int32)
    for data in (t.cuda()[:, :vocab], t[:, :vocab].contiguous().cuda()):
        check(serving.token_logprobs(data, torch.from_numpy(targets).cuda(), top), x, targets, top)


@pytest.mark.parametrize("vocab,top", [(20000, 20), (8191, 32), (50, 32)])
def test_awkward_rows(serving, vocab, top):
    """Equal logits throughout, few distinct values, rising and falling rows, one block of large ones, masks of minus
    infinity and of the lowest number (few or no ids left beside them), zeros of both signs."""
    rng = np.random.default_rng(vocab)
    rows = [np.zeros(vocab), np.full(vocab, -3e38), rng.integers(0, 3, vocab).astype(float), np.arange(vocab) * 1e-3,
            -np.arange(vocab) * 1e-3, np.where((np.arange(vocab) > vocab // 3) & (np.arange(vocab) < vocab // 2), 9.0, 0.0)
            + rng.random(vocab), np.where(rng.random(vocab) < 0.5, -0.0, 0.0)]
    for lowest in (-np.inf, np.finfo(np.float32).min):
        for left in (1, 2, top - 1, top, vocab // 2):
            r = np.full(vocab, lowest)
            at = rng.choice(vocab, left, replace=False)
            r[at] = rng.standard_normal(left) * 5
            rows.append(r)
    x = np.stack(rows).astype(np.float32)
    targets = rng.integers(0, vocab, len(x)).astype(np.int32)
    check(serving.token_logprobs(torch.from_numpy(x).cuda(), torch.from_numpy(targets).cuda(), top), x, targets, top)
    # a row among ordinary ones does not touch them
    y = rng.standard_normal((len(x), vocab)).astype(np.float32)
    y[1::2] = x[1::2]
    check(serving.token_logprobs(torch.from_numpy(y).cuda(), torch.from_numpy(targets).cuda(), top), y, targets, top)


def test_rows_without_a_distribution(serving):
    """NaN, plus infinity, nothing but minus infinity: NaN and no other row's; NaN logits are no alternatives."""
    vocab = 20000
    x = np.random.default_rng(1).standard_normal((6, vocab)).astype(np.float32)
    x[1, 15000] = np.nan
    x[2, 77] = np.inf
    x[3] = -np.inf
    x[4] = np.nan
    x[4, 9000] = 2.0
    targets = np.array([5, 6, 77, 8, 9000, -7], np.int32)
    got = serving.token_logprobs(torch.from_numpy(x).cuda(), torch.from_numpy(targets).cuda(), 8)
    check(got, x, targets, 8, rows=[0, 5])
    lp, entropy, ids, tops = (t.cpu().numpy() for t in got)
    assert np.isnan(lp[1:5]).all() and np.isnan(entropy[1:5]).all() and np.isnan(tops[1:5]).all()
    y = x[1].copy()
    y[15000] = -np.inf
    assert np.array_equal(ids[1], np.lexsort((np.arange(vocab), -y))[:8])
    assert ids[2, 0] == 77 and np.array_equal(ids[3], np.arange(8)) and ids[4].tolist() == [9000] + [-1] * 7


def test_targets(serving):
    """Negative ids are none; ids past the vocabulary give NaN, and an error from the completing form."""
    x = torch.randn(4, 3001, device="cuda")
    targets = torch.tensor([-1, 3001, 2 ** 31 - 1, 3000], dtype=torch.int32, device="cuda")
    got = serving.token_logprobs(x, targets)
    want = torch.log_softmax(x.double(), 1)[3, 3000].item()
    lp = got.logprob.cpu()
    assert lp[0] == 0 and torch.isnan(lp[1:3]).all() and abs(lp[3].item() - want) < 1e-4
    assert got.top_ids.shape == (4, 0) and torch.isfinite(got.entropy).all()
    rt = runtime()
    out = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="out of range"):
        rt.call("tl_token_logprobs", x, 3001, 0, 4, 3001, targets, 0, out, None, None, None)
    targets[1:3] = 0
    rt.call("tl_token_logprobs", x, 3001, 0, 4, 3001, targets, 0, out, None, None, None)
    assert torch.equal(out[[0, 3]], got.logprob[[0, 3]]) and torch.isfinite(out).all()
    rt.close()


def test_refusals(serving):
    x = torch.zeros(2, 100, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: serving.token_logprobs(x.double(), t), lambda: serving.token_logprobs(x.cpu(), t),
                lambda: serving.token_logprobs(x, t.long()), lambda: serving.token_logprobs(x, t[:1]),
                lambda: serving.token_logprobs(x, t, 33), lambda: serving.token_logprobs(x, t, -1),
                lambda: serving.token_logprobs(x[:, :5], t, 6), lambda: serving.token_logprobs(x[:, ::2], t),
                lambda: serving.token_logprobs(x[0], t), lambda: serving.token_logprobs(x[:, :0], t),
                lambda: serving.token_logprobs(x[:1].expand(2, 100), t)):
        with pytest.raises(ValueError):
            bad()
    assert serving.token_logprobs(x[:0], t[:0], 3).top_ids.shape == (0, 3)


def test_graph(serving):
    rng = np.random.default_rng(3)
    x = torch.zeros(3, 20011, device="cuda")
    targets = torch.zeros(3, dtype=torch.int32, device="cuda")
    serving.token_logprobs(x, targets, 9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serving.token_logprobs(x, targets, 9)
    for _ in range(4):
        data, ids = rng.standard_normal((3, 20011)).astype(np.float32), rng.integers(0, 20011, 3).astype(np.int32)
        x.copy_(torch.from_numpy(data))
        targets.copy_(torch.from_numpy(ids))
        graph.replay()
        torch.cuda.synchronize()
        check(got, data, ids, 9)


@pytest.mark.parametrize("dtype,rows,vocab,top", [
    ("f32", 1, 32000, 5), ("bf16", 20, 32000, 32), ("f32", 70, 16001, 20), ("f16", 130, 16385, 3), ("bf16", 300, 16500, 32),
    ("f32", 3, 300007, 0)])
def test_joined_in_place_or_not(serving, dtype, rows, vocab, top):
    """Rows whose parts the last workgroup joins and rows joined by a kernel of their own: a captured call, which has
    no counters, gives the same bits."""
    rng = np.random.default_rng(rows)
    t = torch.from_numpy((rng.standard_normal((rows, vocab)) * 2).astype(np.float32)).to(DT[dtype])
    t[rows // 2, ::3] = 1.5           # more equal logits than a part's room for candidates
    t[rows // 3, 50:] = -float("inf")
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    x, ids = t.cuda(), torch.from_numpy(targets).cuda()
    first = serving.token_logprobs(x, ids, top)
    check(first, t.float().numpy(), targets, top)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = serving.token_logprobs(x, ids, top)
    for _ in range(3):
        graph.replay()
        again = serving.token_logprobs(x, ids, top)
        torch.cuda.synchronize()
        for a, b, c in zip(first, captured, again):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_large_logits(serving):
    """Rows far from zero, on both sides of where the difference to the maximum is taken first."""
    rng = np.random.default_rng(8)
    shifts = [0, 90, -90, 4090, 4101, -4090, -4110, 65504, -1e5, 3e7, -3e7, 1e12, 3.4e38, -3.4e38]
    x = np.stack([rng.standard_normal(9000) * 2 + s for s in shifts]).astype(np.float32)
    targets = rng.integers(0, 9000, len(x)).astype(np.int32)
    check(serving.token_logprobs(torch.from_numpy(x).cuda(), torch.from_numpy(targets).cuda(), 12), x, targets, 12)


def test_engine_score_tokens():
    """A prompt scored by the engine: its tokens' log probabilities are those of the engine's own logits."""
    import oracle
    from lpta.engine import Engine
    cfg = dict(oracle.SMALL_CFG)
    eng = Engine(cfg).load_model(oracle.synthetic_model(cfg, seed=3))
    prompt = np.array([5, 77, 3, 1200, 9, 9, 40], np.int32)
    got = eng.score_tokens(prompt, top=6)
    logits = torch.empty(7, cfg["vocab"], device="cuda")
    eng.rt.call("tl_prefill_logits", 0, prompt, 7, logits)
    targets = np.append(prompt[1:], -1)
    check([torch.from_numpy(got[k]) for k in ("logprob", "entropy", "top_ids", "top_logprobs")], logits.cpu().numpy(), targets, 6)
    assert eng.prefill(prompt)[0] == got["top_ids"][-1, 0]
    eng.close()
