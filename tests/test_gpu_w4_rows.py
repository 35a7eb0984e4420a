"""4-bit projections whose row blocks do not fill the last workgroup row, with exactly the scratch that is asked for."""
from __future__ import annotations

import ctypes as C

import pytest

from gpu_util import runtime, torch as get_torch
from test_gpu_w4 import DT, reference, weights

torch = get_torch()
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,scale,group,m,n,k", [
    ("f32", "f16", 128, 9, 5632, 2048), ("bf16", "bf16", 64, 10, 5632, 2048), ("f32", "f32", 32, 11, 32000, 512),
    ("f16", "f16", 64, 12, 5632, 2048), ("f32", "bf16", 128, 18, 5632, 512), ("bf16", "f16", 64, 100, 5632, 512),
])
def test_row_blocks_to_spare(act, scale, group, m, n, k):
    from lpta import serving
    g = torch.Generator().manual_seed(m + n)
    q, scales = weights(g, n, k, group, scale)
    x = torch.randn(m, k, generator=g).to(DT[act])
    want, tol = reference(x, q, scales, act)
    lin = serving.W4Linear(q.cuda(), scales.cuda())
    xd = x.cuda()
    got = lin(xd)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    # the queueing form, behind its scratch a guard that stays as it is
    need = C.c_int64()
    rt = runtime()
    rt.check(rt.lib.tl_linear_w4_scratch(rt.h, m, k, C.byref(need)))
    block = torch.full((need.value + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(got)
    stream = torch.cuda.current_stream().cuda_stream
    rt.check(rt.lib.tl_linear_w4_async(rt.h, stream, xd.data_ptr(), k, lin_type(act), m, lin.packed.data_ptr(), lin.scale_dtype,
                                       group, n, k, None, 0, y.data_ptr(), n, block.data_ptr(), need.value))
    assert torch.equal(y, got) and (block[need.value:] == 0x5A).all()
    rt.call("tl_linear_w4", xd, k, lin_type(act), m, lin.packed, lin.scale_dtype, group, n, k, None, 0, y.zero_(), n)
    assert torch.equal(y, got)
    rt.close()


def lin_type(act):
    from lpta import _native
    return {"f32": _native.TL_F32, "bf16": _native.TL_BF16, "f16": _native.TL_F16}[act]
