"""Serving operators: a decoding step of many sequences over a paged KV cache.

No counterpart in the reference, whose cache is one dense plane per sequence; the
rotation and the INT8 cache follow its accelerator path (design_decisions A7/B2).

Every call here queues its kernels on torch's current stream of the tensors'
device and returns, as torch's own operations do (the ``_async`` entry points of
include/tl_int8.h): results may be used by later work on that stream, and calls
can be captured into a ``torch.cuda.CUDAGraph`` (but the first on a device).  Scratch
memory is torch's, kept for each stream, and a captured graph has its own, so calls
on different streams and graphs share none; threads may call at the same time.  A
captured call joins the parts of a long row in another order than a queued one does,
so attention may differ between them in the last place.  A ``PagedCache``, ``W4Linear``,
``W8Linear`` or ``W8GatedLinear`` is kept until the calls made with it on other streams than
the one it was made on are done, and as long as a graph that holds such calls.  Tensors are CUDA tensors of one
device; float types are float32, bfloat16 and float16.  Nothing here is differentiable:
results carry no gradient.

What a cache's call finds out of range on the device (a sequence, position or page) it
leaves out; ``PagedCache.check()`` tells.  A token id past the vocabulary gives NaN and is
not reported.  Wrong types, shapes and layouts raise ``TlValueError`` (a ``ValueError``)
at once.
"""
from __future__ import annotations

import ctypes as C
import math
import numbers
import operator
import threading
from typing import NamedTuple

import torch

from . import _native
from ._native import Runtime, TlPagedCache, TlValueError

_ACT = {torch.float32: _native.TL_F32, torch.bfloat16: _native.TL_BF16, torch.float16: _native.TL_F16}
_CACHE = {torch.int8: _native.TL_I8, torch.bfloat16: _native.TL_BF16, torch.float16: _native.TL_F16}
_HANDLES: dict[int, Runtime] = {}
_WORKSPACES: dict[tuple[int, int], "_Workspace"] = {}
_COMPLETING = threading.Lock()   # one call at a time on a handle's own stream


def _runtime(device: torch.device) -> Runtime:
    """The operator handle of a device, made on first use."""
    rt = _HANDLES.get(device.index)
    if rt is None:
        with _COMPLETING, torch.cuda.device(device):
            if device.index in _HANDLES:
                return _HANDLES[device.index]
            if torch._C._cuda_isCurrentStreamCapturing():
                raise _bad("the first call on a device cannot be captured: make it once before")
            rt = Runtime(dict(hidden=64, intermediate=64, n_layers=1, n_heads=1, n_kv_heads=1, head_dim=64, vocab=64,
                              max_pos=64, rms_eps=1e-5, rope_theta=10000.0))
            _HANDLES[device.index] = rt
    return rt


def _stream(dev: torch.device) -> int:
    """The current stream of a device, without the object torch.cuda.current_stream makes."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


class _Workspace:
    """Scratch and zeroed counters of the calls on one stream, which run one after another."""

    def __init__(self, dev: torch.device):
        self.counters = torch.zeros(_native.TL_OP_COUNTERS, dtype=torch.int32, device=dev)
        self.scratch = torch.empty(0, dtype=torch.uint8, device=dev)


def _workspace(dev: torch.device, stream: int, need: int):
    """(scratch address, counters address) for a call on a stream, and what keeps the scratch.
    While the stream is captured the scratch is the graph's own and there are no counters, as
    the graph may run beside other calls."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _workspace(dev, stream, need)
    if torch._C._cuda_isCurrentStreamCapturing():
        own = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        return own.data_ptr() if need else None, None, own
    ws = _WORKSPACES.get((dev.index, stream))
    if ws is None:
        ws = _WORKSPACES.setdefault((dev.index, stream), _Workspace(dev))
    scratch = ws.scratch
    if scratch.shape[0] < need:
        # (the allocator gives the old block to this stream's later work only, and not
        # before another thread's call that holds it is queued)
        scratch = ws.scratch = torch.empty(need + need // 4, dtype=torch.uint8, device=dev)
    return scratch.data_ptr(), ws.counters.data_ptr(), scratch


def _bad(message: str):
    return TlValueError(_native.TL_ERR_BAD_DESCRIPTOR, message)


def _rows(name: str, t, device, width: int | None = None, dtype=None) -> torch.Tensor:
    """A matrix of float rows: elements of a row side by side, any row stride."""
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in _ACT or (dtype and t.dtype != dtype):
        raise _bad(f"{name} must be a {dtype or 'float32, bfloat16 or float16'} tensor on {device}")
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1) or (width is not None and t.shape[1] != width):
        raise _bad(f"{name} must be [rows][{width or 'width'}] with adjacent elements")
    return t


def _ints(name: str, t, device, n: int) -> int:
    """Address of n int32 values side by side."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.dim() != 1:
        raise _bad(f"{name} must be a vector of int32 on {device}")
    if t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise _bad(f"{name} must hold one value for each of {n} rows")
    return t.data_ptr()


def _stride(t) -> int:
    """Elements between rows (one row: any aligned stride will do)."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


class PagedCache:
    """One layer's paged KV cache: pages [n_pages][n_kv_heads][page_size][head_dim] of
    INT8 (with float32 scales per KV head), bfloat16 or float16, and the page table
    [n_seqs][max_pages] int32.  The tensors stay the caller's: pages are handed out by
    writing the table.  ``rope``: cos and sin [positions][head_dim] float32
    (``build_rope_cache``), needed by ``append``.

    Pages of 8 .. 1024 positions (a power of two), heads of 64 or 128.  Page blocks may lie
    in a larger tensor (any stride of the first dimension that keeps 16-byte
    alignment), the table in a wider one.
    """

    def __init__(self, k, v, table, k_scale=None, v_scale=None, rope=None, rt: Runtime | None = None):
        if not isinstance(k, torch.Tensor) or not k.is_cuda or k.dtype not in _CACHE or k.dim() != 4:
            raise _bad("k must be a CUDA tensor [n_pages][n_kv_heads][page_size][head_dim] of int8, bfloat16 or float16")
        dev = k.device
        n_pages, n_kv, page, hd = k.shape
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or t.dtype != k.dtype or t.device != dev or t.shape != k.shape:
                raise _bad("k and v must agree in type, shape and device")
            if t.stride()[1:] != (page * hd, hd, 1) or (n_pages > 1 and t.stride(0) != k.stride(0)):
                raise _bad(f"{name}: the blocks of a page must be dense, and k and v must have one page stride")
        if not isinstance(table, torch.Tensor) or table.dtype != torch.int32 or table.device != dev or table.dim() != 2 \
                or (table.shape[1] > 1 and table.stride(1) != 1):
            raise _bad(f"table must be [n_seqs][max_pages] int32 on {dev} with adjacent entries")
        if (k.dtype == torch.int8) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise _bad("k_scale and v_scale go with an INT8 cache, and only with one")
        for t in (k_scale, v_scale):
            if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev
                                  or t.shape != (n_kv,) or not t.is_contiguous()):
                raise _bad(f"scales must be [n_kv_heads] float32 on {dev}")
        if rope is not None:
            for t in rope:
                if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev or t.dim() != 2 \
                        or t.shape[1] != hd or t.shape != rope[0].shape or not t.is_contiguous():
                    raise _bad(f"rope must be cos and sin [positions][{hd}] float32 on {dev}")
        self.rt = rt or _runtime(dev)
        if self.rt.device != dev.index:
            raise _bad("the handle belongs to another device")
        self.k, self.v, self.table, self.k_scale, self.v_scale, self.rope = k, v, table, k_scale, v_scale, rope
        self.device = dev
        self.n_kv_heads, self.head_dim, self.n_seqs = n_kv, hd, table.shape[0]
        self.fault = torch.zeros(1, dtype=torch.int32, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        self.desc = TlPagedCache(
            ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ptr(table),
            table.stride(0) if table.shape[0] > 1 else table.shape[1], k.stride(0) if n_pages > 1 else n_kv * page * hd,
            _CACHE[k.dtype], n_pages, page, n_kv, hd, table.shape[0], table.shape[1])
        self._desc = C.byref(self.desc)
        self._scratch: dict[tuple[int, int, int], int] = {}
        self._scratch_bytes(0, n_kv)   # the descriptor's own checks

    def _scratch_bytes(self, rows: int, n_heads: int, prefix_len: int = 0) -> int:
        got = self._scratch.get((rows, n_heads, prefix_len))
        if got is None:
            if len(self._scratch) > 4096:   # prefixes of ever new lengths
                self._scratch.clear()
            n = C.c_int64()
            if prefix_len:
                self.rt.check(self.rt.lib.tl_paged_attention_shared_scratch(self.rt.h, self._desc, rows, n_heads, prefix_len,
                                                                            C.byref(n)), "tl_paged_attention_shared_scratch")
            else:
                self.rt.check(self.rt.lib.tl_paged_attention_scratch(self.rt.h, self._desc, rows, n_heads, C.byref(n)),
                              "tl_paged_attention_scratch")
            got = self._scratch[(rows, n_heads, prefix_len)] = n.value
        return got

    def _gain(self, name: str, t):
        """Address of a head's norm gains, or None."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != self.device \
                or t.shape != (self.head_dim,) or not t.is_contiguous():
            raise _bad(f"{name} must be [{self.head_dim}] float32 on {self.device}")
        return t.data_ptr()

    def _row_ids(self, row_seq, row_pos, rows: int):
        if row_seq is None:
            return None, _ints("row_pos", row_pos, self.device, rows)
        return _ints("row_seq", row_seq, self.device, rows), _ints("row_pos", row_pos, self.device, rows)

    def append(self, qkv, row_seq, row_pos, out=None, norm=None, eps: float = 1e-5):
        """Rows of Q|K|V projections [rows][(n_heads + 2 n_kv_heads) * head_dim]: q and k rotated at
        row_pos, k and v written to the cache at row_pos of sequence row_seq (None: row r
        is sequence r; negative: a padded row, skipped).  Returns the rotated q (``out`` if
        given; it may be the q part of qkv); a padded row of a new tensor is undefined.
        ``norm``: gains (q, k), [head_dim] float32 each or None, with which q and k of every
        head are normed first: x / sqrt(mean x^2 + eps) * gain."""
        dev, hd = self.device, self.head_dim
        _rows("qkv", qkv, dev)
        if self.rope is None:
            raise _bad("append needs the cache's rope tables")
        rows, width = qkv.shape
        n_heads = width // hd - 2 * self.n_kv_heads
        if width % hd or n_heads < 0:
            raise _bad("qkv must be [rows][(n_heads + 2 n_kv_heads) * head_dim]")
        seq, pos = self._row_ids(row_seq, row_pos, rows)
        if out is None:
            out = torch.empty((rows, n_heads * hd), dtype=qkv.dtype, device=dev)
        else:
            _rows("out", out, dev, n_heads * hd, qkv.dtype)
            if out.shape[0] != rows:
                raise _bad("out must have a row for each of qkv's")
        if norm is not None:
            try:
                q_gain, k_gain = norm
            except (TypeError, ValueError):
                raise _bad("norm must be the gains of q and of k") from None
            q_gain, k_gain = self._gain("the q gains", q_gain), self._gain("the k gains", k_gain)
            if not isinstance(eps, numbers.Real) or not 0.0 <= eps <= 1e30:
                raise _bad("eps must be a number from 0 on")
        if rows == 0:
            return out
        cos, sin = self.rope
        stride = _stride(qkv)
        q_stride = stride if out.data_ptr() == qkv.data_ptr() and rows == 1 else _stride(out)
        rt = self.rt
        q_out = out.data_ptr() if n_heads else None
        if norm is None:
            st = rt.lib.tl_paged_append_async(
                rt.h, _stream(dev), self._desc, qkv.data_ptr(), stride, _ACT[qkv.dtype],
                rows, n_heads, seq, pos, cos.data_ptr(), sin.data_ptr(), cos.shape[0], q_out, q_stride, self.fault.data_ptr())
        else:
            st = rt.lib.tl_paged_append_norm_async(
                rt.h, _stream(dev), self._desc, qkv.data_ptr(), stride, _ACT[qkv.dtype],
                rows, n_heads, seq, pos, cos.data_ptr(), sin.data_ptr(), cos.shape[0], q_gain, k_gain, eps, q_out, q_stride,
                self.fault.data_ptr())
        if st:
            rt.check(st, "append")
        return out

    def attend(self, q, row_seq, row_pos, scale: float | None = None, out=None):
        """Attention of one query row per token: row r of q [rows][n_heads * head_dim]
        (rotated) over keys 0 .. row_pos[r] of sequence row_seq[r] (None: r); a
        negative position gives zeros, a negative sequence leaves its row of ``out`` as it
        was (undefined in a new tensor).  ``out`` may be q.  ``scale``: 1 / sqrt(head_dim) unless given."""
        return self._attend("attend", q, row_seq, row_pos, 0, 0, scale, out)

    def attend_shared(self, q, row_seq, row_pos, prefix_seq: int, prefix_len: int, scale: float | None = None, out=None):
        """``attend`` of rows whose first ``prefix_len`` positions are those of sequence
        ``prefix_seq``, a prompt that all of them begin with: its keys are read once for all
        rows, key t of row r is position t of prefix_seq for t < prefix_len and of
        row_seq[r] from there on (table entries of row_seq before that are not used).
        Several prompts in a batch: one call each on slices of ``q``, ``row_seq``, ``row_pos``
        and ``out`` where a prompt's rows stand together; into one ``out`` with the other rows'
        row_seq negative also works, but multiplies padded rows as well (4 prompts of 64 rows over
        32768 keys: 366 us by slices, 863).  Worth it for long prompts: up to some 1500 positions
        ``attend`` on tables that hold the prompt's pages is as fast or faster, from some 4000 on
        this is for four rows or more.
        In a captured graph the prefix is the one it was captured with."""
        try:
            prefix_seq, prefix_len = operator.index(prefix_seq), operator.index(prefix_len)
        except TypeError:
            raise _bad("the prefix's sequence and length must be whole numbers") from None
        if not 0 <= prefix_len <= self.desc.max_pages * self.desc.page_size or (
                prefix_len and not 0 <= prefix_seq < self.n_seqs):
            raise _bad("the prefix must lie in the pages of a sequence of the table")
        return self._attend("attend_shared", q, row_seq, row_pos, prefix_seq, prefix_len, scale, out)

    def _attend(self, what, q, row_seq, row_pos, prefix_seq, prefix_len, scale, out):
        dev, hd = self.device, self.head_dim
        _rows("q", q, dev)
        rows, width = q.shape
        n_heads = width // hd
        if width % hd or n_heads == 0 or n_heads % self.n_kv_heads:
            raise _bad("q must be [rows][n_heads * head_dim], n_heads a multiple of the KV heads")
        seq, pos = self._row_ids(row_seq, row_pos, rows)
        if out is None:
            out = torch.empty((rows, width), dtype=q.dtype, device=dev)
        else:
            _rows("out", out, dev, width, q.dtype)
            if out.shape[0] != rows:
                raise _bad("out must have a row for each of q's")
        if rows == 0:
            return out
        need = self._scratch_bytes(rows, n_heads, prefix_len)
        rt, stream = self.rt, _stream(dev)
        scratch, counters, keep = _workspace(dev, stream, need)
        scale = 1.0 / math.sqrt(hd) if scale is None else scale
        if prefix_len:
            st = rt.lib.tl_paged_attention_shared_async(
                rt.h, stream, self._desc, q.data_ptr(), _stride(q), _ACT[q.dtype], rows, n_heads, seq, pos, prefix_seq,
                prefix_len, scale, out.data_ptr(), _stride(out), scratch, need, counters, self.fault.data_ptr())
        else:
            st = rt.lib.tl_paged_attention_async(
                rt.h, stream, self._desc, q.data_ptr(), _stride(q), _ACT[q.dtype], rows, n_heads, seq, pos, scale,
                out.data_ptr(), _stride(out), scratch, need, counters, self.fault.data_ptr())
        if st:
            rt.check(st, what)
        return out

    def check(self) -> None:
        """Wait for the cache's calls on the current stream and raise if one of them met a
        sequence, position or page out of range."""
        if int(self.fault.item()):
            self.fault.zero_()
            raise _bad("a sequence, position or page is out of range")


def quantize_w4(w, group: int = 128, scale_dtype=torch.float16, rt: Runtime | None = None):
    """4-bit weights of float32 ones [n][k] (tl_quantize_w4_rows): (q, scales) for ``W4Linear``."""
    if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dtype != torch.float32 or w.dim() != 2:
        raise _bad("w must be a CUDA tensor [n][k] of float32")
    if scale_dtype not in _ACT:
        raise _bad("scales are float32, bfloat16 or float16")
    n, k = w.shape
    if group not in (32, 64, 128) or k == 0 or k % group:
        raise _bad("group must be 32, 64 or 128 and divide k")
    rt = rt or _runtime(w.device)
    if rt.device != w.device.index:
        raise _bad("the handle belongs to another device")
    q = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, k // group), dtype=scale_dtype, device=w.device)
    with _COMPLETING:
        rt.call("tl_quantize_w4_rows", w.contiguous(), n, k, group, _ACT[scale_dtype], q, scales)
    return q, scales


class W4Linear:
    """A projection with 4-bit weights: y = x w^T (+ residual), w[n][k] = q[n][k] *
    scales[n][k // group].  q [n][k / 2] uint8 holds two weights of -8 .. 7 (two's
    complement) in a byte, the even column in the low nibble; scales [n][k / group] are
    float32, bfloat16 or float16; group is 32, 64 or 128.  Both are packed here, once, into
    the order the kernels read, and not kept.  x is taken to 2^-30 of the largest of each
    128 of its columns (tl_linear_w4)."""

    def __init__(self, q, scales, rt: Runtime | None = None):
        if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype != torch.uint8 or q.dim() != 2 or not q.is_contiguous():
            raise _bad("q must be a contiguous CUDA tensor [n][k / 2] of uint8")
        if not isinstance(scales, torch.Tensor) or scales.device != q.device or scales.dtype not in _ACT \
                or scales.dim() != 2 or scales.shape[0] != q.shape[0] or not scales.is_contiguous():
            raise _bad(f"scales must be contiguous [n][k / group] float32, bfloat16 or float16 on {q.device}")
        self.device = q.device
        self.n, self.k = q.shape[0], 2 * q.shape[1]
        if scales.shape[1] == 0 or self.k % scales.shape[1]:
            raise _bad("scales must hold one value for each group of a row")
        self.group = self.k // scales.shape[1]
        self.scale_dtype = _ACT[scales.dtype]
        self.rt = rt = rt or _runtime(q.device)
        if rt.device != q.device.index:
            raise _bad("the handle belongs to another device")
        n = C.c_int64()
        rt.check(rt.lib.tl_w4_packed_bytes(rt.h, self.n, self.k, self.group, self.scale_dtype, C.byref(n)), "W4Linear")
        self.packed = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        with _COMPLETING:
            rt.call("tl_pack_w4", q, scales, self.scale_dtype, self.group, self.n, self.k, self.packed)
        self._scratch: dict[int, int] = {}

    @classmethod
    def from_float(cls, w, group: int = 128, scale_dtype=torch.float16, rt: Runtime | None = None) -> "W4Linear":
        """Quantize and pack float32 weights [n][k]."""
        return cls(*quantize_w4(w, group, scale_dtype, rt), rt)

    def _scratch_bytes(self, rows: int) -> int:
        got = self._scratch.get(rows)
        if got is None:
            n = C.c_int64()
            self.rt.check(self.rt.lib.tl_linear_w4_scratch(self.rt.h, rows, self.k, C.byref(n)), "tl_linear_w4_scratch")
            got = self._scratch[rows] = n.value
        return got

    def __call__(self, x, residual=None, out=None):
        """x [rows][k] -> [rows][n] in x's type; ``out`` may be ``residual``, not x."""
        dev = self.device
        _rows("x", x, dev, self.k)
        rows = x.shape[0]
        if out is None:
            out = torch.empty((rows, self.n), dtype=x.dtype, device=dev)
        else:
            _rows("out", out, dev, self.n, x.dtype)
        if residual is not None:
            _rows("residual", residual, dev, self.n, x.dtype)
        if out.shape[0] != rows or (residual is not None and residual.shape[0] != rows):
            raise _bad("out and residual must have a row for each of x's")
        if rows == 0:
            return out
        need = self._scratch_bytes(rows)
        rt, stream = self.rt, _stream(dev)
        scratch, _, keep = _workspace(dev, stream, need)
        st = rt.lib.tl_linear_w4_async(
            rt.h, stream, x.data_ptr(), _stride(x), _ACT[x.dtype], rows, self.packed.data_ptr(), self.scale_dtype,
            self.group, self.n, self.k, None if residual is None else residual.data_ptr(),
            0 if residual is None else _stride(residual), out.data_ptr(), _stride(out), scratch, need)
        if st:
            rt.check(st, "W4Linear")
        return out


def quantize_w8(w, rt: Runtime | None = None):
    """8-bit weights of float32 ones [n][k] (tl_quantize_weight_rows): (q int8, scales
    [n] float32) for ``W8Linear`` and ``W8GatedLinear``."""
    if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dtype != torch.float32 or w.dim() != 2 or 0 in w.shape:
        raise _bad("w must be a CUDA tensor [n][k] of float32")
    rt = rt or _runtime(w.device)
    if rt.device != w.device.index:
        raise _bad("the handle belongs to another device")
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    scales = torch.empty(w.shape[0], dtype=torch.float32, device=w.device)
    with _COMPLETING:
        rt.call("tl_quantize_weight_rows", w.contiguous(), w.shape[0], w.shape[1], q, scales)
    return q, scales


class _W8:
    """Packed 8-bit weights, of one projection or of a gate and an up projection."""

    def __init__(self, pairs, rt: Runtime | None):
        q = pairs[0][0]
        for w, s in pairs:
            if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dtype != torch.int8 or w.dim() != 2 \
                    or not w.is_contiguous() or w.shape != q.shape or w.device != q.device:
                raise _bad("weights must be contiguous CUDA tensors [n][k] of int8, of one shape and device")
            if not isinstance(s, torch.Tensor) or s.device != q.device or s.dtype != torch.float32 \
                    or s.shape != (q.shape[0],) or not s.is_contiguous():
                raise _bad(f"scales must be [n] float32 on {q.device}")
        self.device = q.device
        self.n, self.k = q.shape
        self.gated = len(pairs) == 2
        self.rt = rt = rt or _runtime(q.device)
        if rt.device != q.device.index:
            raise _bad("the handle belongs to another device")
        n = C.c_int64()
        rt.check(rt.lib.tl_w8_packed_bytes(rt.h, self.n, self.k, int(self.gated), C.byref(n)), type(self).__name__)
        self.packed = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        with _COMPLETING:
            rt.call("tl_pack_w8", *pairs[0], *(pairs[1] if self.gated else (None, None)), self.n, self.k, self.packed)
        self._scratch: dict[int, int] = {}

    def _scratch_bytes(self, rows: int) -> int:
        got = self._scratch.get(rows)
        if got is None:
            n = C.c_int64()
            self.rt.check(self.rt.lib.tl_linear_w8_scratch(self.rt.h, rows, self.k, C.byref(n)), "tl_linear_w8_scratch")
            got = self._scratch[rows] = n.value
        return got

    def _call(self, x, residual, out):
        dev = self.device
        _rows("x", x, dev, self.k)
        rows = x.shape[0]
        if out is None:
            out = torch.empty((rows, self.n), dtype=x.dtype, device=dev)
        else:
            _rows("out", out, dev, self.n, x.dtype)
        if residual is not None:
            _rows("residual", residual, dev, self.n, x.dtype)
        if out.shape[0] != rows or (residual is not None and residual.shape[0] != rows):
            raise _bad("out and residual must have a row for each of x's")
        if rows == 0:
            return out
        need = self._scratch_bytes(rows)
        rt, stream = self.rt, _stream(dev)
        scratch = keep = None
        if need:
            scratch, _, keep = _workspace(dev, stream, need)
        st = rt.lib.tl_linear_w8_async(
            rt.h, stream, x.data_ptr(), _stride(x), _ACT[x.dtype], rows, self.packed.data_ptr(), int(self.gated), self.n,
            self.k, None if residual is None else residual.data_ptr(), 0 if residual is None else _stride(residual),
            out.data_ptr(), _stride(out), scratch, need)
        if st:
            rt.check(st, type(self).__name__)
        return out


class W8Linear(_W8):
    """A projection in 8-bit integers: y = x w^T (+ residual), with w[n][k] = q[n][k] *
    scales[n] and each row of x quantized on the way, x8 = rne(x / s), s = max |x| / 127.
    q [n][k] int8 and scales [n] float32 (``quantize_w8``) are packed here, once, and not
    kept.  Any n and any k up to 2^17; sums are exact (tl_linear_w8)."""

    def __init__(self, q, scales, rt: Runtime | None = None):
        super().__init__([(q, scales)], rt)

    @classmethod
    def from_float(cls, w, rt: Runtime | None = None) -> "W8Linear":
        """Quantize and pack float32 weights [n][k]."""
        return cls(*quantize_w8(w, rt), rt)

    def __call__(self, x, residual=None, out=None):
        """x [rows][k] -> [rows][n] in x's type; ``out`` may be ``residual``, not x."""
        return self._call(x, residual, out)


class W8GatedLinear(_W8):
    """The first half of a gated feed-forward block in 8-bit integers, in one product:
    y = silu(x gate^T) * (x up^T), both projections as ``W8Linear``'s."""

    def __init__(self, gate, gate_scales, up, up_scales, rt: Runtime | None = None):
        super().__init__([(gate, gate_scales), (up, up_scales)], rt)

    @classmethod
    def from_float(cls, gate, up, rt: Runtime | None = None) -> "W8GatedLinear":
        """Quantize and pack float32 weights [n][k]."""
        return cls(*quantize_w8(gate, rt), *quantize_w8(up, rt), rt)

    def __call__(self, x, out=None):
        """x [rows][k] -> [rows][n] in x's type; ``out`` is apart from x."""
        return self._call(x, None, out)


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor        # [rows] float32
    entropy: torch.Tensor        # [rows] float32, nats
    top_ids: torch.Tensor        # [rows][top] int32
    top_logprobs: torch.Tensor   # [rows][top] float32


_LOGPROBS_SCRATCH: dict[tuple[int, int, int], int] = {}


def token_logprobs(logits, targets, top: int = 0, rt: Runtime | None = None) -> TokenLogprobs:
    """Of each row of logits [rows][vocab]: the log probability of targets[row] (int32; negative:
    none, 0; an id past the vocabulary gives NaN), the entropy, and the ``top`` (up to 32)
    most probable ids, the lower one first among equal logits."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise _bad("logits must be a CUDA tensor")
    dev = logits.device
    _rows("logits", logits, dev)
    rows, vocab = logits.shape
    ids = _ints("targets", targets, dev, rows)
    if not 0 <= top <= min(32, vocab) or vocab == 0:
        raise _bad("top must be 0 .. 32 and at most the vocabulary")
    logprob, entropy = torch.empty((2, rows), dtype=torch.float32, device=dev).unbind()
    best = torch.empty((rows, top), dtype=torch.int32, device=dev)
    best_lp = torch.empty((rows, top), dtype=torch.float32, device=dev)
    got = TokenLogprobs(logprob, entropy, best, best_lp)
    if rows == 0:
        return got
    rt = rt or _runtime(dev)
    if rt.device != dev.index:
        raise _bad("the handle belongs to another device")
    need = _LOGPROBS_SCRATCH.get((rows, vocab, top))
    if need is None:
        n = C.c_int64()
        rt.check(rt.lib.tl_token_logprobs_scratch(rt.h, rows, vocab, top, C.byref(n)), "tl_token_logprobs_scratch")
        need = _LOGPROBS_SCRATCH[(rows, vocab, top)] = n.value
    stream = _stream(dev)
    scratch, counters, keep = _workspace(dev, stream, need)
    st = rt.lib.tl_token_logprobs_async(
        rt.h, stream, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab,
        _ACT[logits.dtype], rows, vocab, ids, top, logprob.data_ptr(), entropy.data_ptr(),
        best.data_ptr(), best_lp.data_ptr(), scratch, need, counters, None)
    if st:
        rt.check(st, "token_logprobs")
    return got
