"""A layer's steps of a padded batch of conversations that begin with one prompt, made of the serving operators together:
8-bit Q|K|V projection, append with norms, attention over the shared prompt, 8-bit O projection onto the residual, gated
8-bit projections, 8-bit down projection onto the residual.  The prompt's rows go through the same calls first; pages
are handed out as conversations grow.  Every stage against its definition in 64 bits on what the stage before gave."""
from __future__ import annotations

import math

import pytest

from gpu_util import torch as get_torch
from test_gpu_append_norm import normed, rotated, tables
from test_gpu_w8 import STEP, TINY, U, close, product, silu_bound

torch = get_torch()
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}


@pytest.mark.parametrize("act,cache", [("f32", "i8"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("captured", [False, True])
def test_steps(act, cache, captured):
    from lpta import serving
    heads, kv, hd, d, ffn, page, plen, steps = 8, 2, 64, 448, 1000, 16, 75, 6
    b, live = 5, [1, 2, 3, 4, -1]                          # the last row pads the batch
    g = torch.Generator().manual_seed(21)

    def weights(n, k):
        return serving.quantize_w8(torch.randn(n, k, generator=g).cuda() / math.sqrt(k))
    sets = {"qkv": weights((heads + 2 * kv) * hd, d), "o": weights(d, heads * hd), "gate": weights(ffn, d),
            "up": weights(ffn, d), "down": weights(d, ffn)}
    qkv, o, down = (serving.W8Linear(*sets[n]) for n in ("qkv", "o", "down"))
    glu = serving.W8GatedLinear(*sets["gate"], *sets["up"])
    host = {n: (q.cpu(), s.cpu()) for n, (q, s) in sets.items()}
    gains = [(1 + 0.2 * torch.randn(hd, generator=g)) for _ in range(2)]
    norm = tuple(t.cuda() for t in gains)
    cos, sin = tables(128, hd)
    scales = [torch.full((kv,), 0.04, device="cuda") for _ in range(2)] if cache == "i8" else [None, None]
    pool = [torch.zeros(40, kv, page, hd, dtype=DT[cache], device="cuda") for _ in range(2)]
    table = torch.full((5, 7), -1, dtype=torch.int32, device="cuda")
    c = serving.PagedCache(*pool, table, *scales, rope=(cos.cuda(), sin.cuda()))
    free = list(range(39, -1, -1))
    for p in range(-(-plen // page)):
        table[0, p] = free.pop()
    whole = plen // page                                   # the conversations have the prompt's whole pages
    table[1:, :whole] = table[0, :whole]

    def layer(x, seq, pos, n):
        y = qkv(x)
        q = c.append(y, seq, pos, norm=norm, eps=1e-6)
        a = c.attend_shared(q, seq, pos, 0, n)
        z = o(a, residual=x)
        f = glu(z)
        return y, q, a, z, f, down(f, residual=z)

    def values(which, seq, n, own_from):
        """Keys or values 0 .. n - 1 that a row of the sequence attends, [n][kv][hd] float64."""
        t, s = ((c.k, scales[0]), (c.v, scales[1]))[which]
        rows = [t[int(table[0 if p < own_from else seq, p // page]), :, p % page] for p in range(n)]
        x = torch.stack(rows).cpu().double()
        return x if s is None else x * s.cpu().double()[:, None]

    def check(x, seq, pos, n, got):
        y, q, a, z, f, out = (t.cpu() for t in got)
        x = x.cpu()
        rows = [i for i, s in enumerate(seq) if s >= 0]
        want, tol = product(x, *host["qkv"])
        close(y[rows], want[rows], tol[rows], act)
        xf = y.float().view(len(x), heads + 2 * kv, hd).numpy()
        cs, sn = cos.numpy()[pos], sin.numpy()[pos]
        wq = torch.from_numpy(rotated(normed(xf[:, :heads], gains[0].numpy(), 1e-6), cs, sn)).to(DT[act]).reshape(len(x), -1)
        assert torch.equal(q[rows], wq[rows])
        wk = torch.from_numpy(rotated(normed(xf[:, heads:heads + kv], gains[1].numpy(), 1e-6), cs, sn))
        for t, w, s in ((c.k, wk, scales[0]), (c.v, torch.from_numpy(xf[:, heads + kv:]), scales[1])):
            if s is not None:
                w = torch.round(w / s.cpu()[:, None]).clamp(-127, 127)
            for i in rows:
                assert torch.equal(t[int(table[seq[i], pos[i] // page]), :, pos[i] % page].cpu(), w[i].to(DT[cache]))
        for i in rows:
            k, v = (values(w, seq[i], pos[i] + 1, n) for w in (0, 1))
            for h in range(heads):
                kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
                qh = q[i, h * hd:(h + 1) * hd].double()
                p = torch.softmax(kh @ qh / 8, 0)
                mag = (kh.abs() @ qh.abs()).max().item() / 8
                # scores, probabilities and sums as in the attention's own test
                t = (2 * (((hd + 12) * U + 2.0 ** -21) * mag * 1.4427 + 2.0 ** -22) + 2.0 ** -14 + 2 * (2 * len(kh) + 80) * U) * (p @ vh.abs())
                w = p @ vh
                assert ((a[i, h * hd:(h + 1) * hd].double() - w).abs() <= t + STEP[act] * (w.abs() + t) + TINY[act]).all()
        for got_y, name, src, res in ((z, "o", a, x), (out, "down", f, z)):
            want, tol = product(src, *host[name])
            want = want + res.double()
            close(got_y[rows], want[rows], (tol + U * (want.abs() + tol))[rows], act)
        want, tol = silu_bound(*product(z, *host["gate"]), *product(z, *host["up"]))
        close(f[rows], want[rows], tol[rows], act)

    # the prompt: its rows attend its own keys up to theirs
    ids = [torch.zeros(plen, dtype=torch.int32, device="cuda"), torch.arange(plen, dtype=torch.int32, device="cuda")]
    x = torch.randn(plen, d, generator=g).to(DT[act]).cuda()
    check(x, [0] * plen, list(range(plen)), 0, layer(x, *ids, 0))
    got = layer(x, *ids, plen)                             # and the same as rows of a shared prefix
    check(x, [0] * plen, list(range(plen)), plen, got)

    own = [9, 1, 30, 16]                                   # keys that the conversations have of their own already
    for s, n in enumerate(own, 1):
        for p in range(whole, (plen + n) // page + 1):
            table[s, p] = free.pop()
        ids = [torch.full((n,), s, dtype=torch.int32, device="cuda"),
               torch.arange(plen, plen + n, dtype=torch.int32, device="cuda")]
        layer(torch.randn(n, d, generator=g).to(DT[act]).cuda(), *ids, plen)
    x = torch.zeros(b, d, dtype=DT[act], device="cuda")
    seq = torch.tensor(live, dtype=torch.int32, device="cuda")
    pos = torch.tensor([plen + n for n in own] + [0], dtype=torch.int32, device="cuda")
    if captured:
        layer(x, seq, pos, plen)                           # warm; rewritten by the first step
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, seq, pos, plen)
    for i in range(steps):
        at = [plen + n + i for n in own] + [0]
        for s in range(1, 5):
            if int(table[s, at[s - 1] // page]) < 0:
                table[s, at[s - 1] // page] = free.pop()
        x.copy_(torch.randn(b, d, generator=g).to(DT[act]))
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        if captured:
            graph.replay()
            got = out
        else:
            got = layer(x, seq, pos, plen)
        torch.cuda.synchronize()
        check(x, live, at, plen, got)
    c.check()


def test_threads_and_streams():
    """Threads that call at the same time, on streams of their own and on one they share, with sizes that make the
    shared workspace grow: every call gives what it gives alone."""
    import threading
    from lpta import serving
    g = torch.Generator().manual_seed(2)
    lin = serving.W8Linear(*serving.quantize_w8(torch.randn(256, 512, generator=g).cuda()))
    w = torch.randn(96, 512, generator=g).cuda()
    k, v = (torch.randn(130, 2, 16, 64, generator=g).half().cuda() for _ in range(2))
    table = torch.arange(130, dtype=torch.int32, device="cuda").view(2, 65)
    cache = serving.PagedCache(k, v, table)
    jobs = []
    for n in range(4):
        x = torch.randn(3 + 90 * n, 512, generator=g).cuda()
        q = torch.randn(2 + 20 * n, 512, generator=g).cuda()
        seq = torch.ones(len(q), dtype=torch.int32, device="cuda")
        pos = 700 + 10 * torch.arange(len(q), dtype=torch.int32, device="cuda") % 300

        def job(x=x, q=q, seq=seq, pos=pos, n=n):
            pair = serving.W8GatedLinear.from_float(w, w)
            return [lin(x), pair(x), cache.attend_shared(q, seq, pos, 0, 500 + n)]
        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    common = torch.cuda.Stream()
    for alone in (False, True):
        got, errors = [[] for _ in jobs], []

        def work(n):
            try:
                stream = torch.cuda.Stream() if alone else common
                with torch.cuda.stream(stream):
                    for _ in range(15):
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
                assert all(torch.equal(a, b) for a, b in zip(again, want[n])), (alone, n)
    cache.check()
