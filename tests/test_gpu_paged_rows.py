"""Attention over the paged cache with as many rows as a prompt has, joined by a kernel of its own."""
from __future__ import annotations

import pytest

from gpu_util import torch as get_torch

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,rows", [(12, 12, 1500), (20, 2, 700), (32, 4, 2000), (9, 1, 65)])
def test_prompt_rows_captured(heads, kv, rows):
    """Causal rows of one prompt, some padded and one of them at the end of a long sequence, in a captured call: as the
    call that joins in place, and as 64 bits say."""
    from lpta import serving
    g = torch.Generator().manual_seed(rows)
    page, hd, longest = 16, 64, 9000
    need = [-(-rows // page), -(-longest // page)]
    k, v = (torch.randn(sum(need), kv, page, hd, generator=g).half().cuda() for _ in range(2))
    table = torch.zeros(2, max(need), dtype=torch.int32)
    table[0, :need[0]] = torch.arange(need[0])
    table[1] = need[0] + torch.arange(need[1])
    c = serving.PagedCache(k, v, table.cuda())
    seq, pos = [0] * rows, list(range(rows))
    for r in range(7, rows, 31):
        seq[r] = -1
    seq[rows // 2], pos[rows // 2] = 1, longest - 1
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    q = torch.randn(rows, heads * hd, generator=g).cuda()
    eager = c.attend(q, *ids, out=torch.zeros_like(q))
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(q, *ids, out=out)
    for _ in range(3):
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(rows):
            if seq[r] < 0:
                assert (out[r] == 3.0).all()
                out[r] = eager[r]
        # the same parts in another order: float32 sums of at most 512 of them
        assert (out - eager).abs().max() <= 512 * 2.0 ** -24 * 4
    c.check()
    # rows in 64 bits
    for r in (0, 1, rows // 2, rows - 1):
        n = pos[r] + 1
        kd, vd = (t[c.table[seq[r], :-(-n // page)].long()].transpose(1, 2).reshape(-1, kv, hd)[:n].double() for t in (k, v))
        for h in range(heads):
            p = torch.softmax(kd[:, h * kv // heads] @ q[r].double().view(heads, hd)[h] / 8, 0)
            assert (out[r].double().view(heads, hd)[h] - p @ vd[:, h * kv // heads]).abs().max() < 2e-5
