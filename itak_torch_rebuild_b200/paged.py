"""The paged cache: rotation, append and attention over pages, on torch tensors.

``PagedKv`` names a pair of page pools the caller owns; ``append`` stores a ragged batch's new rows (K rotated on the
way) and ``attention`` attends them.  ``rope_table`` makes a rotation's frequencies, plain or scaled for long contexts,
and ``rope_apply`` rotates rows on their own, forward or as a gradient.  Every call queues work on the current stream of
the tensors' device (or on ``stream``, a handle), allocates nothing on the device but a default ``out`` (of the stream that
writes it, as torch counts it) and, once per stream, a workspace, and raises :class:`CudaComputeError` with the library's text
when it is refused.  Tensors that a call on ``stream`` shares with other streams are the caller's to order, as in torch.

No gradient passes through these calls: while gradients are enabled they refuse tensors that require one (``rope_apply`` with
``inverse=True`` is the rotation's gradient, for a backward pass of the caller's).  What they write counts as written in place,
so that autograd notices when a backward pass still wants the old values.

A batch: sequence ``s`` owns the packed rows ``[row_start[s], row_start[s + 1])`` and ``kv_len[s]`` keys, its new rows
included; the key of position ``p`` is row ``p % page_size`` of page ``table[s][p // page_size]``.  ``table``,
``row_start`` and ``kv_len`` are int32 tensors on the device, read when the work runs, so a captured graph follows them.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .backend import CudaComputeError

_ROW_DTYPES = {torch.float32: _lib.ROW_F32, torch.float16: _lib.ROW_F16, torch.bfloat16: _lib.ROW_BF16}
_SCALINGS = {"plain": _lib.ROPE_PLAIN, "linear": _lib.ROPE_LINEAR, "base": _lib.ROPE_BASE, "bands": _lib.ROPE_BANDS,
             "ramp": _lib.ROPE_RAMP, "pairs": _lib.ROPE_PAIRS}
_ERROR_LEN = 256

# A decode step's kernels run for a few microseconds, so the descriptors are packed in one go (filling a ctypes structure
# takes six times as long); the layouts are those of _lib's structures.
_PACK_ROPE = struct.Struct("8Q6I2if4x").pack
_PACK_BATCH = struct.Struct("4Q4I").pack
_PACK_APPEND = struct.Struct("9Q3Iif4x").pack
_PACK_ATTENTION = struct.Struct("7Q3Iif4x").pack
_OUT_OF_RANGE = (struct.error, OverflowError)  # a value that its field cannot hold
for _s, _f in ((_lib.RopeDesc, "8Q6I2if4x"), (_lib.PagedBatch, "4Q4I"), (_lib.PagedAppendDesc, "9Q3Iif4x"),
               (_lib.PagedAttentionDesc, "7Q3Iif4x")):
    assert C.sizeof(_s) == struct.calcsize(_f), _s

_calls: dict = {}


def _entry(name: str, descriptors: int):
    """The library's entry point taking packed descriptors, looked up once (``_calls``)."""
    fn = _lib.load()[name]
    fn.restype = C.c_int
    fn.argtypes = [C.c_char_p] * descriptors + [C.c_void_p, C.c_void_p, C.c_size_t]
    _calls[name] = fn
    return fn


def _refuse(msg: str, code: int = _lib.ERR_INVALID_ARGUMENT):
    raise CudaComputeError(code, msg)


class _Reason(threading.local):
    """A thread's buffer for the reason of a refusal, handed to every call (by its address, which is what a call costs least
    with): a call is made once, whatever it returns."""

    def __init__(self):
        self.text = C.create_string_buffer(_ERROR_LEN)
        self.at = C.addressof(self.text)

    def refuse(self, rc: int):
        raise CudaComputeError(rc, self.text.value.decode("utf-8", "replace"))


_reason = _Reason()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


# Handles with a meaning of their own: the default stream (two names), and "the calling thread's", one handle for many streams.
_DEFAULT_STREAMS = (0, 1)
_PER_THREAD_STREAM = 2


def _stream_object(device: int, stream: int):
    """The torch stream of a handle."""
    if stream in _DEFAULT_STREAMS:
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(stream, device=device)


def _capturing(device: int, stream: int) -> bool:
    """Whether ``stream`` of ``device`` is being captured, the current stream or not (the default one never is)."""
    if stream in _DEFAULT_STREAMS:
        return False
    if device == torch.cuda.current_device() and stream == _raw_stream(device):
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(_stream_object(device, stream)):
        return torch.cuda.is_current_stream_capturing()


def _new_rows(shape, dtype, device: int, stream: Optional[int]) -> torch.Tensor:
    """Memory for a result of a call on ``stream`` (``None``: the current one).  It has to be the allocator's memory of that
    stream: a block of another stream's may still be read there by work queued before it was freed, and may be handed out
    again there while ``stream`` writes it."""
    if stream == _PER_THREAD_STREAM:  # one handle, a stream for every thread: the allocator could not tell them apart
        _refuse("a call on the per-thread default stream needs its result's memory given")
    if stream is None or stream == _raw_stream(device):
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(_stream_object(device, stream)):
        return torch.empty(shape, dtype=dtype, device=device)


# Counts tensors as written to, for autograd's check of what it has saved.
_written = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


_grad_enabled = torch.is_grad_enabled


def _no_gradient():
    _refuse("no gradient passes through this call: detach its tensors, or call it under torch.no_grad()")


def _rows(t: torch.Tensor, what: str, rows: int, heads: int, head_dim: int, dtype, device: int) -> int:
    """The row stride of a ``[rows][heads][head_dim]`` tensor whose heads are contiguous (of a single row: torch gives it any)."""
    if t.dtype is not dtype or t.get_device() != device:
        _refuse(f"{what} must be {dtype} on device {device}, got {t.dtype} on {t.device}")
    if t.shape != (rows, heads, head_dim):
        _refuse(f"{what} has shape {tuple(t.shape)}, expected {(rows, heads, head_dim)}")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != head_dim and heads > 1):
        _refuse(f"the heads of {what} must be contiguous, got strides {(s0, s1, s2)}")
    return s0 if rows > 1 else heads * head_dim


def _vector(t: torch.Tensor, what: str, dtype, n: Optional[int], device: int) -> int:
    """The address of a contiguous vector of ``n`` elements (any number: ``None``)."""
    if t.dtype is not dtype or t.get_device() != device:
        _refuse(f"{what} must be {dtype} on device {device}, got {t.dtype} on {t.device}")
    if t.dim() != 1 or (n is not None and t.numel() != n) or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous vector{'' if n is None else f' of {n} elements'}, got {tuple(t.shape)}")
    return t.data_ptr()


def rope_table(rotary_dim: int, base: float, *, scaling: str = "plain", factor: float = 1.0, original_context: float = 0.0,
               low: float = 1.0, high: float = 0.0, pair_factors: Optional[Sequence[float]] = None, magnitude: float = 0.0):
    """The frequencies of a rotation: ``(inv_freq, magnitude)``, an f64 array of ``rotary_dim / 2`` angles per position and
    the factor on sine and cosine (``itk_rope_table``).  ``scaling``: ``plain``, ``linear``, ``base``, ``bands``, ``ramp`` (turns
    ``low`` < ``high`` over ``original_context``) or ``pairs`` (``pair_factors``); all of these are f32 values, the table is f64.
    Copy it to the device once."""
    if scaling not in _SCALINGS:
        _refuse(f"rope: unknown scaling {scaling!r}")
    pf = None
    if pair_factors is not None:
        pf = np.ascontiguousarray(np.asarray(pair_factors, dtype=np.float32))
        if pf.size != max(rotary_dim, 0) // 2:
            raise CudaComputeError(_lib.ERR_SHAPE_MISMATCH, f"pair_factors: got {pf.size}, expected {rotary_dim // 2}")
    if not 0 <= rotary_dim <= 0xffffffff:
        _refuse("rope: rotary_dim must be even, >= 2, and <= head_dim")
    cfg = _lib.RopeConfig(pf.ctypes.data_as(C.POINTER(C.c_float)) if pf is not None else None, rotary_dim, _SCALINGS[scaling],
                          base, factor, original_context, low, high, magnitude)
    out = np.empty(max(rotary_dim // 2, 1), dtype=np.float64)
    mag, err = C.c_float(), C.create_string_buffer(_ERROR_LEN)
    rc = _lib.load().itk_rope_table(C.byref(cfg), out.ctypes.data, C.byref(mag), err, _ERROR_LEN)
    if rc != _lib.OK:
        _refuse(err.value.decode("utf-8", "replace"), rc)
    return out, mag.value


def rope_apply(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, pairing: int = 0, magnitude: float = 1.0,
               inverse: bool = False, out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Rotates ``x`` ``[rows][heads][head_dim]`` (f32, f16 or bf16; any row and head strides), row ``r`` at
    ``positions[r]`` (int32, read as unsigned: there are no positions before 0).  ``pairing`` 0 joins channels (2i, 2i + 1), 1 joins (i, i + rotary_dim / 2), with
    ``rotary_dim = 2 * len(inv_freq)``; ``inverse=True`` maps the gradient of the result to the gradient of ``x``.
    ``out`` may be ``x``.  At least one row and head."""""
    dtype, dev = _ROW_DTYPES.get(x.dtype), x.get_device()
    if dtype is None or dev < 0 or x.dim() != 3:
        _refuse(f"x must be an f32, f16 or bf16 [rows][heads][head_dim] tensor on a CUDA device, got {x.dtype} {tuple(x.shape)} on {x.device}")
    if _grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
        _no_gradient()
    shape, given = x.shape, out is not None
    if out is None:
        out = _new_rows(shape, x.dtype, dev, stream)
    elif out.dtype is not x.dtype or out.get_device() != dev or out.shape != shape:
        _refuse(f"out must be {x.dtype} {tuple(shape)} on {x.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
    rows, heads, head_dim = shape
    at = _vector(positions, "positions", torch.int32, rows, dev)
    table = _vector(inv_freq, "inv_freq", torch.float64, None, dev)
    x0, x1, x2 = x.stride()
    o0, o1, o2 = out.stride()
    if x2 != 1 or o2 != 1:
        _refuse("the channels of x and out must be contiguous")
    try:
        d = _PACK_ROPE(x.data_ptr(), out.data_ptr(), at, table, x0, x1, o0, o1, rows, heads, head_dim, 2 * inv_freq.numel(), pairing,
                       1 if inverse else 0, dtype, dev, magnitude)
    except _OUT_OF_RANGE as e:
        _refuse(f"an argument is out of range: {e}")
    rc = (_calls.get("itk_rope_apply") or _entry("itk_rope_apply", 1))(d, _raw_stream(dev) if stream is None else stream, _reason.at, _ERROR_LEN)
    if rc != _lib.OK:
        _reason.refuse(rc)
    if given:
        _written([out])
    return out


_workspaces: dict = {}


def attention_workspace(device) -> torch.Tensor:
    """A workspace for ``PagedKv.attention`` calls on ``device``, cleared.  Calls that may run at the same time - on two
    streams, or from two graphs that are replayed on two streams - need one each.  Make it before a capture begins."""
    device = torch.device(device)
    n = _lib.load().itk_paged_attention_workspace(device.index or 0)
    if n == 0:
        raise CudaComputeError(_lib.ERR_CUDA, f"no workspace for {device}: the device cannot be used")
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():  # its clearing would become part of the graph, its memory the graph's
            _refuse("a workspace cannot be made while the current stream is being captured")
        ws = torch.zeros(n, dtype=torch.uint8, device=device)
        torch.cuda.current_stream().synchronize()  # whatever stream uses it first
    return ws


def release_workspaces():
    """Gives up this module's own workspaces (39 MB for every stream that has called without one), once their devices have
    come to rest.  Later calls make new ones."""
    for device in {device for device, _ in _workspaces}:
        torch.cuda.synchronize(device)
    _workspaces.clear()


def wait_limit(kclocks: int = 0):
    """Bounds the waits inside the tensor-core kernel, in units of 1024 SM clocks (0: about a second;
    ``itk_paged_attention_wait_limit``).  Where one runs out, rows come out as NaN and bit 4 of ``status`` is raised."""
    if not 0 <= kclocks <= 0xffffffff or _lib.load().itk_paged_attention_wait_limit(kclocks) != _lib.OK:
        _refuse(f"the bound of a wait is 0..2^22 x 1024 clocks, got {kclocks}")


class PagedKv:
    """A pair of page pools: ``k`` and ``v`` 4-dimensional f16 or bf16 tensors of the same shape and strides,
    ``[pages][kv_heads][page_size][head_dim]`` with ``layout="head"`` or ``[pages][page_size][kv_heads][head_dim]`` with
    ``layout="token"``.  The pools stay the caller's; this object only describes them."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, *, layout: str = "head"):
        if layout not in ("head", "token"):
            _refuse(f"layout is 'head' or 'token', got {layout!r}")
        # a dimension of one element is never stepped over, and torch gives it any stride
        steps = [[s if n > 1 else 0 for n, s in zip(x.shape, x.stride())] for x in (k, v)]
        if k.dim() != 4 or k.shape != v.shape or steps[0] != steps[1]:
            _refuse(f"the pools must be two 4-dimensional tensors of one shape and one set of strides, got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.device.type != "cuda" or k.dtype not in (torch.float16, torch.bfloat16):
            _refuse(f"the pools must be f16 or bf16 tensors on a CUDA device, got {k.dtype} on {k.device}")
        if v.device != k.device or v.dtype is not k.dtype:
            _refuse(f"the pools must be of one type on one device, got {k.dtype} on {k.device} and {v.dtype} on {v.device}")
        st = steps[0]
        if st[3] != 1 and k.shape[3] > 1:
            _refuse("the channels of a page must be contiguous")
        self.k, self.v, self.layout, self.device, self.dtype = k, v, layout, k.device, k.dtype
        heads_at, rows_at = (1, 2) if layout == "head" else (2, 1)
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape[0], k.shape[heads_at], k.shape[rows_at], k.shape[3]
        self._index = k.get_device()
        self._scale = 1.0 / math.sqrt(max(self.head_dim, 1))
        if max(k.shape) > 0xffffffff:  # (a ctypes field would cut it)
            _refuse(f"the pools' shape {tuple(k.shape)} is out of range")
        self._kv = bytes(_lib.PagedKv(k.data_ptr(), v.data_ptr(), st[0], st[heads_at], st[rows_at], self.n_pages, self.page_size,
                                      self.kv_heads, self.head_dim, _ROW_DTYPES[k.dtype], self._index))

    def _batch(self, table, row_start, kv_len, total_rows, status) -> bytes:
        dev, n, i32 = self._index, kv_len.numel(), torch.int32
        # one test of what is right; what is wrong is looked for afterwards
        if (kv_len.dtype is not i32 or row_start.dtype is not i32 or table.dtype is not i32 or kv_len.get_device() != dev
                or row_start.get_device() != dev or table.get_device() != dev or kv_len.dim() != 1 or row_start.dim() != 1
                or table.dim() != 2 or row_start.numel() != n + 1 or not kv_len.is_contiguous() or not row_start.is_contiguous()):
            _vector(kv_len, "kv_len", i32, None, dev)
            _vector(row_start, "row_start", i32, n + 1, dev)
            _refuse(f"table must be {i32} [{n}][pages of a sequence] on device {dev}, got {table.dtype} {tuple(table.shape)} on {table.device}")
        rows, width = table.shape
        stride, inner = table.stride()
        if rows != n or (inner != 1 and width > 1):
            _refuse(f"table must be [{n}][pages of a sequence] with contiguous rows, got {(rows, width)}")
        word = 0
        if status is not None:
            word = _vector(status, "status", i32, None, dev)
            if status.numel() < 1:
                _refuse("status must hold one element")
        try:
            return _PACK_BATCH(table.data_ptr(), row_start.data_ptr(), kv_len.data_ptr(), word, n, width, stride if n > 1 else width, total_rows)
        except _OUT_OF_RANGE as e:
            _refuse(f"a size of the batch is out of range: {e}")

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, *,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
               pairing: int = 0, magnitude: float = 1.0, status: Optional[torch.Tensor] = None, stream: Optional[int] = None):
        """Stores the new rows ``k``, ``v`` ``[rows][kv_heads][head_dim]`` into their pages, K rotated by ``inv_freq``
        (``None``: stored as it is), and returns ``q`` rotated alike (in ``q_out``, which may be ``q``) when ``q`` is
        given.  f32 rows go into f16 pages, 16-bit rows into pages of their type (``itk_paged_append``)."""
        dev, d, dtype = self._index, self.head_dim, k.dtype
        row_dtype = _ROW_DTYPES.get(dtype)
        if row_dtype is None or k.dim() != 3:
            _refuse(f"rows must be f32, f16 or bf16 [rows][{self.kv_heads}][{d}], got {dtype} {tuple(k.shape)}")
        if _grad_enabled() and (k.requires_grad or v.requires_grad or self.k.requires_grad or self.v.requires_grad
                                or (q is not None and q.requires_grad) or (q_out is not None and q_out.requires_grad)):
            _no_gradient()
        rows = k.shape[0]
        k_row = _rows(k, "k", rows, self.kv_heads, d, dtype, dev)
        v_row = _rows(v, "v", rows, self.kv_heads, d, dtype, dev)
        q_row = q_out_row = q_heads = q_at = q_out_at = 0
        if q is not None:
            if q.dim() != 3:
                _refuse(f"q has shape {tuple(q.shape)}, expected [{rows}][heads][{d}]")
            q_heads = q.shape[1]
            q_row = _rows(q, "q", rows, q_heads, d, dtype, dev)
            if q_out is None:
                q_out = _new_rows((rows, q_heads, d), dtype, dev, stream)
            q_out_row = _rows(q_out, "q_out", rows, q_heads, d, dtype, dev)
            q_at, q_out_at = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            _refuse("q, q_out and q_heads go together")
        freq = rotary = 0
        if inv_freq is not None:
            freq, rotary = _vector(inv_freq, "inv_freq", torch.float64, None, dev), 2 * inv_freq.numel()
        batch = self._batch(table, row_start, kv_len, rows, status)
        if rows == 0:  # torch gives empty tensors no address
            return q_out
        try:
            a = _PACK_APPEND(q_at, q_out_at, k.data_ptr(), v.data_ptr(), freq, q_row, q_out_row, k_row, v_row, q_heads, rotary, pairing,
                             row_dtype, magnitude)
        except _OUT_OF_RANGE as e:
            _refuse(f"an argument is out of range: {e}")
        rc = (_calls.get("itk_paged_append") or _entry("itk_paged_append", 3))(self._kv, batch, a, _raw_stream(dev) if stream is None else stream, _reason.at, _ERROR_LEN)
        if rc != _lib.OK:
            _reason.refuse(rc)
        _written([self.k, self.v] if q_out is None else [self.k, self.v, q_out])
        return q_out

    def attention(self, q: torch.Tensor, table: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, *, max_rows: int,
                  scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
        """Causal grouped-query attention of the rows ``q`` ``[rows][q_heads][head_dim]`` over their sequences' pages,
        within ``window`` keys when it is not 0 (``itk_paged_attention``).  ``max_rows`` bounds the rows of one sequence
        and only chooses between kernels; ``scale`` is ``1 / sqrt(head_dim)`` unless given; ``lse`` ``[rows][q_heads]``
        f32 receives the log-sum-exp.  Without ``workspace`` calls of one stream share one of this module's; a call
        that is being captured, or that runs on the per-thread default stream, must be given its own
        (``attention_workspace``).  A stream that is destroyed is to be synchronised first: its handle, and the workspace
        that goes with it, may become another stream's."""
        dev, d, dtype = self._index, self.head_dim, q.dtype
        row_dtype = _ROW_DTYPES.get(dtype)
        if row_dtype is None or q.dim() != 3:
            _refuse(f"rows must be f32, f16 or bf16 [rows][heads][{d}], got {dtype} {tuple(q.shape)}")
        if _grad_enabled() and (q.requires_grad or self.k.requires_grad or self.v.requires_grad
                                or (out is not None and out.requires_grad) or (lse is not None and lse.requires_grad)):
            _no_gradient()
        rows, q_heads, _ = q.shape
        q_row = _rows(q, "q", rows, q_heads, d, dtype, dev)
        if out is None:
            out = _new_rows((rows, q_heads, d), dtype, dev, stream)
        out_row = _rows(out, "out", rows, q_heads, d, dtype, dev)
        lse_at = 0
        if lse is not None:
            if lse.dtype is not torch.float32 or lse.get_device() != dev or lse.shape != (rows, q_heads) or not lse.is_contiguous():
                _refuse(f"lse must be a contiguous {torch.float32} [{rows}][{q_heads}] tensor on device {dev}, got {lse.dtype} {tuple(lse.shape)} on {lse.device}")
            lse_at = lse.data_ptr()
        stream = _raw_stream(dev) if stream is None else stream
        if workspace is None:
            if stream == _PER_THREAD_STREAM:  # one handle, a stream for every thread
                _refuse("a call on the per-thread default stream needs a workspace of its own (attention_workspace)")
            if _capturing(dev, stream):
                _refuse("a call that is being captured needs a workspace of its own (attention_workspace)")
            workspace = _workspaces.get((dev, stream))
            if workspace is None:
                workspace = _workspaces[(dev, stream)] = attention_workspace(self.device)
        elif workspace.dtype is not torch.uint8 or workspace.get_device() != dev or not workspace.is_contiguous():
            _refuse(f"the workspace must be a contiguous {torch.uint8} tensor on device {dev}, got {workspace.dtype} on {workspace.device}")
        batch = self._batch(table, row_start, kv_len, rows, status)
        if rows == 0:  # torch gives empty tensors no address
            return out
        try:
            a = _PACK_ATTENTION(q.data_ptr(), out.data_ptr(), lse_at, workspace.data_ptr(), workspace.numel(), q_row, out_row, q_heads,
                                max_rows, window, row_dtype, self._scale if scale is None else scale)
        except _OUT_OF_RANGE as e:
            _refuse(f"an argument is out of range: {e}")
        rc = (_calls.get("itk_paged_attention") or _entry("itk_paged_attention", 3))(self._kv, batch, a, stream, _reason.at, _ERROR_LEN)
        if rc != _lib.OK:
            _reason.refuse(rc)
        _written([out] if lse is None else [out, lse])
        return out
