"""Decoding steps of a padded batch made of the serving operators together, as a server makes them: 4-bit Q|K|V
projection, append with rotation, attention over the paged cache, 4-bit O projection onto the residual, 4-bit head,
log probabilities of the chosen tokens; pages handed out as sequences grow.  Against the same steps in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import torch as get_torch
from test_gpu_w4 import dense

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cache,tol", [("f32", "f16", 2e-3), ("bf16", "bf16", 6e-2), ("f32", "i8", 6e-2)])
@pytest.mark.parametrize("captured", [False, True])
def test_steps(act, cache, tol, captured):
    """The tolerance is the cache's rounding of keys and values (half steps 2^-11, 2^-8, and half of one of 127
    levels: at most 2^-8 of the largest) or the activations', each carried through products that do not enlarge it
    (gain-free random weights), for the logits of standard deviation 1 that the head makes."""
    from lpta import serving, build_rope_cache
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
    heads, kv, hd, d, vocab, page, b, steps = 8, 2, 64, 512, 1000, 16, 5, 20
    g = torch.Generator().manual_seed(11)
    start = [14, 0, 31, 5, 0]
    live = [0, 1, 2, 3, -1]                       # the last row pads the batch

    weights = [serving.quantize_w4(torch.randn(n, k, generator=g).cuda() / math.sqrt(k), 64, torch.float16)
               for n, k in (((heads + 2 * kv) * hd, d), (d, heads * hd), (vocab, d))]
    wqkv, wo, head = (serving.W4Linear(*p) for p in weights)
    w = [dense(q.cpu(), s.cpu()) for q, s in weights]
    cos, sin = (torch.from_numpy(t) for t in build_rope_cache(128, hd, 10000.0))
    k = torch.zeros(24, kv, page, hd, dtype=dt[cache], device="cuda")
    table = torch.full((4, 5), -1, dtype=torch.int32, device="cuda")
    scales = [torch.full((kv,), 0.04, device="cuda") for _ in range(2)] if cache == "i8" else [None, None]
    c = serving.PagedCache(k, torch.zeros_like(k), table, *scales, rope=(cos.cuda(), sin.cuda()))
    free = list(range(23, -1, -1))

    past = [(torch.randn(n, kv, hd, generator=g), torch.randn(n, kv, hd, generator=g)) for n in start[:4]]
    for s, (pk, pv) in enumerate(past):
        for j in range(start[s]):
            if j % page == 0:
                table[s, j // page] = free.pop()
            for t, p in ((c.k, pk), (c.v, pv)):
                row = p[j] if cache != "i8" else (p[j] / 0.04).round().clamp(-127, 127)
                t[int(table[s, j // page]), :, j % page] = row.to(dt[cache]).cuda()
    hist = [[list(pk.double()), list(pv.double())] for pk, pv in past]

    x = torch.zeros(b, d, dtype=dt[act], device="cuda")
    seq = torch.tensor(live, dtype=torch.int32, device="cuda")
    pos = torch.tensor(start, dtype=torch.int32, device="cuda")
    chosen = torch.zeros(b, dtype=torch.int32, device="cuda")
    att = torch.zeros(b, heads * hd, dtype=dt[act], device="cuda")

    def step():
        q = c.append(wqkv(x), seq, pos)
        c.attend(q, seq, pos, out=att)
        logits = head(wo(att, residual=x))
        return logits, serving.token_logprobs(logits, chosen, top=4)

    if captured:
        for s in range(4):
            table[s, start[s] // page] = int(table[s, start[s] // page]) if start[s] % page else free[-1]
        step()                                    # warm; rewritten by the first step
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
    worst = 0.0
    for i in range(steps):
        xs = torch.randn(b, d, generator=g).to(dt[act])
        ids = torch.randint(0, vocab, (b,), generator=g, dtype=torch.int32)
        for s in range(4):
            if (start[s] + i) % page == 0:
                table[s, (start[s] + i) // page] = free.pop()
        x.copy_(xs)
        pos.copy_(torch.tensor(start, dtype=torch.int32) + i)
        chosen.copy_(ids)
        if captured:
            graph.replay()
            logits, got = out
        else:
            logits, got = step()
        torch.cuda.synchronize()
        for s in range(4):
            xd = xs[s].double()
            y = w[0] @ xd
            p = start[s] + i
            qk = y[:(heads + kv) * hd].view(-1, hd)
            turned = torch.cat([-qk[:, hd // 2:], qk[:, :hd // 2]], 1)
            qk = qk * cos[p].double() + turned * sin[p].double()
            hist[s][0].append(qk[heads:])
            hist[s][1].append(y[(heads + kv) * hd:].view(kv, hd))
            kk, vv = (torch.stack(h) for h in hist[s])
            o = torch.cat([torch.softmax(kk[:, h // 4] @ qk[h] / 8, 0) @ vv[:, h // 4] for h in range(heads)])
            z = w[2] @ (xd + w[1] @ o)
            worst = max(worst, (logits[s].cpu().double() - z).abs().max().item())
            lp = torch.log_softmax(logits[s].double(), 0)
            assert abs(got.logprob[s].item() - lp[ids[s]].item()) < 1e-4
            top = np.lexsort((np.arange(vocab), -logits[s].float().cpu().numpy()))[:4]
            assert got.top_ids[s].tolist() == top.tolist()
        assert torch.isfinite(logits).all() and (att[4] == 0).all()
    c.check()
    assert worst < tol, worst


def test_threads_and_streams():
    """Threads that call at the same time, on streams of their own and on one they share, with sizes that make the
    shared workspace grow: every call gives what it gives alone."""
    import threading
    from lpta import serving
    g = torch.Generator().manual_seed(2)
    lin = serving.W4Linear(*serving.quantize_w4(torch.randn(256, 512, generator=g).cuda()))
    k, v = (torch.randn(260, 1, 16, 64, generator=g).half().cuda() for _ in range(2))
    table = torch.arange(260, dtype=torch.int32, device="cuda").view(2, 130)
    cache = serving.PagedCache(k, v, table)
    dense_w = torch.randn(96, 512, generator=g).cuda()
    jobs = []
    for n in range(4):
        x = torch.randn(3 + 5 * n, 512, generator=g).cuda()
        logits = torch.randn(4 + 9 * n, 20000 + 7777 * n, generator=g).cuda()
        ids = torch.randint(0, 20000, (len(logits),), generator=g, dtype=torch.int32).cuda()
        q = torch.randn(1 + n, 256, generator=g).cuda()
        seq = torch.arange(1 + n, dtype=torch.int32, device="cuda") % 2
        pos = torch.full((1 + n,), 900 + 300 * n, dtype=torch.int32, device="cuda")

        def job(x=x, logits=logits, ids=ids, q=q, seq=seq, pos=pos, n=n):
            made = serving.W4Linear.from_float(dense_w, 64)
            return [lin(x), made(x), *serving.token_logprobs(logits, ids, 3 * n), cache.attend(q, seq, pos)]
        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    for own in (False, True):
        got, errors = [[] for _ in jobs], []

        def work(n):
            try:
                stream = torch.cuda.Stream() if own else shared
                with torch.cuda.stream(stream):
                    for _ in range(20):
                        got[n].append(jobs[n]())
                stream.synchronize()
            except Exception as e:   # noqa: BLE001
                errors.append(e)
        threads = [threading.Thread(target=work, args=(n,)) for n in range(len(jobs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for n in range(len(jobs)):
            for again in got[n]:
                assert all(torch.equal(a, b) for a, b in zip(again, want[n])), (own, n)
    cache.check()


def test_first_call_is_not_captured(monkeypatch):
    """The call that would make a device's handle is refused while its stream is captured."""
    from lpta import serving
    x = torch.randn(2, 100, device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    want = serving.token_logprobs(x, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with monkeypatch.context() as m:
            m.setattr(serving, "_HANDLES", {})
            with pytest.raises(ValueError, match="captured"):
                serving.token_logprobs(x, ids)
        got = serving.token_logprobs(x, ids)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.logprob, want.logprob)
