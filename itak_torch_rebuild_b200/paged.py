"""The paged cache: rotation, append and attention over pages, on torch tensors.

``PagedKv`` names a pair of page pools the caller owns; ``append`` stores a ragged batch's new rows (K rotated on the
way) and ``attention`` attends them.  ``rope_table`` makes a rotation's frequencies, plain or scaled for long contexts,
and ``rope_apply`` rotates rows on their own, forward or as a gradient.  Every call queues work on the current stream of
the tensors' device (or on ``stream``), allocates nothing on the device but a default ``out`` and, once per stream, a
workspace, and raises :class:`CudaComputeError` with the library's text when it is refused.

A batch: sequence ``s`` owns the packed rows ``[row_start[s], row_start[s + 1])`` and ``kv_len[s]`` keys, its new rows
included; the key of position ``p`` is row ``p % page_size`` of page ``table[s][p // page_size]``.  ``table``,
``row_start`` and ``kv_len`` are int32 tensors on the device, read when the work runs, so a captured graph follows them.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .backend import CudaComputeError

_ROW_DTYPES = {torch.float32: _lib.ROW_F32, torch.float16: _lib.ROW_F16, torch.bfloat16: _lib.ROW_BF16}
_SCALINGS = {"plain": _lib.ROPE_PLAIN, "linear": _lib.ROPE_LINEAR, "base": _lib.ROPE_BASE, "bands": _lib.ROPE_BANDS,
             "ramp": _lib.ROPE_RAMP, "pairs": _lib.ROPE_PAIRS}
_ERROR_LEN = 256


def _refuse(msg: str):
    raise CudaComputeError(_lib.ERR_INVALID_ARGUMENT, msg)


def _raise(rc: int, err):
    raise CudaComputeError(rc, err.value.decode("utf-8", "replace"))


def _on(t: torch.Tensor, device: torch.device, what: str, dtype=None):
    if t.device != device or (dtype is not None and t.dtype is not dtype):
        _refuse(f"{what} must be {'a tensor' if dtype is None else dtype} on {device}, got {t.dtype} on {t.device}")


def _stream(device: torch.device, stream: Optional[int]) -> int:
    return torch.cuda.current_stream(device).cuda_stream if stream is None else stream


def _heads(t: torch.Tensor, what: str, heads: Optional[int], head_dim: int, rows: Optional[int] = None):
    """A ``[rows][heads][head_dim]`` tensor whose heads are contiguous; returns its row stride."""
    if t.dim() != 3 or t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads) or (rows is not None and t.shape[0] != rows):
        _refuse(f"{what} has shape {tuple(t.shape)}, expected [{'rows' if rows is None else rows}][{heads or 'heads'}][{head_dim}]")
    st = t.stride()
    if st[2] != 1 or (t.shape[1] > 1 and st[1] != head_dim):
        _refuse(f"the heads of {what} must be contiguous, got strides {st}")
    return st[0]


def rope_table(rotary_dim: int, base: float, *, scaling: str = "plain", factor: float = 1.0, original_context: float = 0.0,
               low: float = 1.0, high: float = 0.0, pair_factors: Optional[Sequence[float]] = None, magnitude: float = 0.0):
    """The frequencies of a rotation: ``(inv_freq, magnitude)``, an f64 array of ``rotary_dim / 2`` angles per position and
    the factor on sine and cosine (``itk_rope_table``).  ``scaling``: ``plain``, ``linear``, ``base``, ``bands``, ``ramp`` (turns
    ``low`` < ``high`` over ``original_context``) or ``pairs`` (``pair_factors``).  Copy the table to the device once."""
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
        _raise(rc, err)
    return out, mag.value


def rope_apply(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, pairing: int = 0, magnitude: float = 1.0,
               inverse: bool = False, out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Rotates ``x`` ``[rows][heads][head_dim]`` (f32, f16 or bf16; any row and head strides), row ``r`` at
    ``positions[r]`` (int32).  ``pairing`` 0 joins channels (2i, 2i + 1), 1 joins (i, i + rotary_dim / 2), with
    ``rotary_dim = 2 * len(inv_freq)``; ``inverse=True`` maps the gradient of the result to the gradient of ``x``.
    ``out`` may be ``x``."""
    dev = x.device
    if dev.type != "cuda" or x.dtype not in _ROW_DTYPES or x.dim() != 3:
        _refuse(f"x must be an f32, f16 or bf16 [rows][heads][head_dim] tensor on a CUDA device, got {x.dtype} {tuple(x.shape)} on {dev}")
    rows, heads, head_dim = x.shape
    if out is None:
        out = torch.empty((rows, heads, head_dim), dtype=x.dtype, device=dev)
    else:
        _on(out, dev, "out", x.dtype)
        if out.shape != x.shape:
            _refuse(f"out has shape {tuple(out.shape)}, expected {tuple(x.shape)}")
    _on(positions, dev, "positions", torch.int32)
    _on(inv_freq, dev, "inv_freq", torch.float64)
    if positions.shape != (rows,) or not positions.is_contiguous():
        _refuse(f"positions must be a contiguous [{rows}] tensor, got {tuple(positions.shape)}")
    if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        _refuse("inv_freq must be a contiguous vector")
    xs, os = x.stride(), out.stride()
    if (xs[2] != 1 or os[2] != 1) and head_dim > 1:
        _refuse("the channels of x and out must be contiguous")
    d = _lib.RopeDesc(x.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), xs[0], xs[1], os[0], os[1],
                      rows, heads, head_dim, 2 * inv_freq.shape[0], pairing, 1 if inverse else 0, _ROW_DTYPES[x.dtype],
                      dev.index, magnitude)
    err = C.create_string_buffer(_ERROR_LEN)
    rc = _lib.load().itk_rope_apply(C.byref(d), _stream(dev, stream), err, _ERROR_LEN)
    if rc != _lib.OK:
        _raise(rc, err)
    return out


_workspaces: dict = {}


def attention_workspace(device) -> torch.Tensor:
    """A workspace for ``PagedKv.attention`` calls on ``device``, cleared.  Calls that may run at the same time - on two
    streams, or from two graphs that are replayed on two streams - need one each."""
    device = torch.device(device)
    n = _lib.load().itk_paged_attention_workspace(device.index or 0)
    if n == 0:
        raise CudaComputeError(_lib.ERR_CUDA, f"no workspace for {device}: the device cannot be used")
    with torch.cuda.device(device):
        ws = torch.zeros(n, dtype=torch.uint8, device=device)
        torch.cuda.current_stream().synchronize()  # whatever stream uses it first
    return ws


class PagedKv:
    """A pair of page pools: ``k`` and ``v`` 4-dimensional f16 or bf16 tensors of the same shape and strides,
    ``[pages][kv_heads][page_size][head_dim]`` with ``layout="head"`` or ``[pages][page_size][kv_heads][head_dim]`` with
    ``layout="token"``.  The pools stay the caller's; this object only describes them."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, *, layout: str = "head"):
        if layout not in ("head", "token"):
            _refuse(f"layout is 'head' or 'token', got {layout!r}")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride():
            _refuse(f"the pools must be two 4-dimensional tensors of one shape and one set of strides, got {tuple(k.shape)} and {tuple(v.shape)}")
        if k.device.type != "cuda" or k.dtype not in (torch.float16, torch.bfloat16):
            _refuse(f"the pools must be f16 or bf16 tensors on a CUDA device, got {k.dtype} on {k.device}")
        _on(v, k.device, "v", k.dtype)
        st = k.stride()
        if st[3] != 1:
            _refuse("the channels of a page must be contiguous")
        self.k, self.v, self.layout, self.device, self.dtype = k, v, layout, k.device, k.dtype
        heads_at, rows_at = (1, 2) if layout == "head" else (2, 1)
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape[0], k.shape[heads_at], k.shape[rows_at], k.shape[3]
        self._lib = _lib.load()
        self._kv = _lib.PagedKv(k.data_ptr(), v.data_ptr(), st[0], st[heads_at], st[rows_at], self.n_pages, self.page_size,
                                self.kv_heads, self.head_dim, _ROW_DTYPES[k.dtype], k.device.index)

    def _batch(self, table, row_start, kv_len, total_rows, status):
        dev = self.device
        n = kv_len.shape[0]
        for t, what in ((table, "table"), (row_start, "row_start"), (kv_len, "kv_len")):
            _on(t, dev, what, torch.int32)
        if table.dim() != 2 or table.shape[0] != n or (table.stride(1) != 1 and table.shape[1] > 1):
            _refuse(f"table must be [{n}][pages of a sequence] with contiguous rows, got {tuple(table.shape)}")
        if row_start.shape != (n + 1,) or kv_len.dim() != 1 or not row_start.is_contiguous() or not kv_len.is_contiguous():
            _refuse(f"row_start must be a contiguous [{n + 1}] and kv_len a contiguous [{n}] tensor, got {tuple(row_start.shape)} and {tuple(kv_len.shape)}")
        if status is not None:
            _on(status, dev, "status", torch.int32)
            if status.numel() < 1:
                _refuse("status must hold one element")
        return _lib.PagedBatch(table.data_ptr(), row_start.data_ptr(), kv_len.data_ptr(),
                               None if status is None else status.data_ptr(), n, table.shape[1], table.stride(0), total_rows)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, *,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
               pairing: int = 0, magnitude: float = 1.0, status: Optional[torch.Tensor] = None, stream: Optional[int] = None):
        """Stores the new rows ``k``, ``v`` ``[rows][kv_heads][head_dim]`` into their pages, K rotated by ``inv_freq``
        (``None``: stored as it is), and returns ``q`` rotated alike (in ``q_out``, which may be ``q``) when ``q`` is
        given.  f32 rows go into f16 pages, 16-bit rows into pages of their type (``itk_paged_append``)."""
        dev, d = self.device, self.head_dim
        rows = k.shape[0]
        k_row = _heads(k, "k", self.kv_heads, d)
        v_row = _heads(v, "v", self.kv_heads, d, rows)
        _on(k, dev, "k")
        if k.dtype not in _ROW_DTYPES:
            _refuse(f"rows must be f32, f16 or bf16, got {k.dtype}")
        _on(v, dev, "v", k.dtype)
        q_row = q_out_row = q_heads = 0
        if q is not None:
            _on(q, dev, "q", k.dtype)
            q_row, q_heads = _heads(q, "q", None, d, rows), q.shape[1]
            if q_out is None:
                q_out = torch.empty((rows, q_heads, d), dtype=q.dtype, device=dev)
            _on(q_out, dev, "q_out", k.dtype)
            q_out_row = _heads(q_out, "q_out", q_heads, d, rows)
        elif q_out is not None:
            _refuse("q, q_out and q_heads go together")
        if inv_freq is not None:
            _on(inv_freq, dev, "inv_freq", torch.float64)
            if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
                _refuse("inv_freq must be a contiguous vector")
        batch = self._batch(table, row_start, kv_len, rows, status)
        a = _lib.PagedAppendDesc(None if q is None else q.data_ptr(), None if q is None else q_out.data_ptr(), k.data_ptr(),
                                 v.data_ptr(), None if inv_freq is None else inv_freq.data_ptr(), q_row, q_out_row, k_row, v_row,
                                 q_heads, 0 if inv_freq is None else 2 * inv_freq.shape[0], pairing, _ROW_DTYPES[k.dtype], magnitude)
        if rows == 0:  # torch gives empty tensors no address
            return q_out
        err = C.create_string_buffer(_ERROR_LEN)
        rc = self._lib.itk_paged_append(C.byref(self._kv), C.byref(batch), C.byref(a), _stream(dev, stream), err, _ERROR_LEN)
        if rc != _lib.OK:
            _raise(rc, err)
        return q_out

    def attention(self, q: torch.Tensor, table: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, *, max_rows: int,
                  scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
        """Causal grouped-query attention of the rows ``q`` ``[rows][q_heads][head_dim]`` over their sequences' pages,
        within ``window`` keys when it is not 0 (``itk_paged_attention``).  ``max_rows`` bounds the rows of one sequence
        and only chooses between kernels; ``scale`` is ``1 / sqrt(head_dim)`` unless given; ``lse`` ``[rows][q_heads]``
        f32 receives the log-sum-exp.  Without ``workspace`` calls of one stream share one of this module's; a call
        that is being captured must be given its own (``attention_workspace``)."""
        dev, d = self.device, self.head_dim
        rows, q_heads = q.shape[0], q.shape[1]
        q_row = _heads(q, "q", None, d)
        _on(q, dev, "q")
        if q.dtype not in _ROW_DTYPES:
            _refuse(f"rows must be f32, f16 or bf16, got {q.dtype}")
        if out is None:
            out = torch.empty((rows, q_heads, d), dtype=q.dtype, device=dev)
        else:
            _on(out, dev, "out", q.dtype)
        out_row = _heads(out, "out", q_heads, d, rows)
        if lse is not None:
            _on(lse, dev, "lse", torch.float32)
            if lse.shape != (rows, q_heads) or not lse.is_contiguous():
                _refuse(f"lse must be a contiguous [{rows}][{q_heads}] tensor, got {tuple(lse.shape)}")
        if not 0 <= window <= 0xffffffff or not 0 <= max_rows <= 0xffffffff:
            _refuse(f"window {window} and max_rows {max_rows} must not be negative")
        raw = _stream(dev, stream)
        if workspace is None:
            workspace = _workspaces.get((dev.index, raw))
            if torch.cuda.is_current_stream_capturing():
                _refuse("a call that is being captured needs a workspace of its own (attention_workspace)")
            if workspace is None:
                workspace = _workspaces[(dev.index, raw)] = attention_workspace(dev)
        else:
            _on(workspace, dev, "workspace", torch.uint8)
            if not workspace.is_contiguous():
                _refuse("the workspace must be contiguous")
        batch = self._batch(table, row_start, kv_len, rows, status)
        if rows == 0:  # torch gives empty tensors no address
            return out
        a = _lib.PagedAttentionDesc(q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), workspace.data_ptr(),
                                    workspace.numel(), q_row, out_row, q_heads, max_rows, window, _ROW_DTYPES[q.dtype],
                                    1.0 / math.sqrt(d) if scale is None else scale)
        err = C.create_string_buffer(_ERROR_LEN)
        rc = self._lib.itk_paged_attention(C.byref(self._kv), C.byref(batch), C.byref(a), raw, err, _ERROR_LEN)
        if rc != _lib.OK:
            _raise(rc, err)
        return out
