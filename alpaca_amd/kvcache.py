"""KV caches on the device, held in 4 bits or in pages, and the operators around them.

``Q4Cache`` owns one layer's cache (``ahip_kv_q4_*``, ``ahip_attention_q4`` of
include/alpaca_hip.h) and the attention's workspace; ``qk_norm_rope`` is the
per-head norm of queries and keys with their rotation.  ``PagedCache`` owns one
layer's f16 cache in pages (``ahip_paged_*``), ``PagedBatch`` describes a step of
many sequences over it.  Rows, outputs, gains
and tables are device addresses (``ahip_malloc``, or any allocator of the same
device), rows [tokens][heads][head_dim] of ``dtype`` "f32" or "f16" with
``stride`` elements from one token to the next (None: dense).  Work is queued on
``stream`` (a handle of ``ahip_stream_create``; None: the context's stream), in
order and without waiting.
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from . import _lib as L
from .model import HIPContext, _LIVE

DTYPE = {"f32": L.F32, "f16": L.F16}
WORKSPACE_ZERO = 2048  # AHIP_Q4_WORKSPACE_ZERO
PAGED_WORKSPACE_ZERO = 4096  # AHIP_PAGED_WORKSPACE_ZERO
# ahip_norm_rope's bytes (L.NormRopeC), packed in a third of the time that the structure's 21 fields take
_NORM_ROPE = struct.Struct("@PPPqqPPPqqPPiiiiiiiif4x").pack

# ahip_paged_rows's bytes (L.PagedRowsC)
_PAGED_ROWS = struct.Struct("@PPPPqqqqPiiii").pack


class Q4Cache:
    """Keys and values of up to ``capacity`` tokens, Q4_0 blocks along the head dimension."""

    def __init__(self, context: HIPContext, kv_heads: int, capacity: int, head_dim: int):
        lib, n = L.lib(), C.c_int64()
        L.check(lib.ahip_kv_q4_bytes(kv_heads, capacity, head_dim, C.byref(n)))
        self.context, self.kv_heads, self.capacity, self.head_dim = context, kv_heads, capacity, head_dim
        self.bytes = 2 * n.value
        self._desc = L.KVQ4C(None, None, kv_heads, head_dim, capacity)
        self._cache = C.byref(self._desc)
        self._width = kv_heads * head_dim
        self._store, self._load, self._attention = lib.ahip_kv_q4_store, lib.ahip_kv_q4_load, lib.ahip_attention_q4
        self._work, self._work_bytes, self._reserved = None, 0, set()
        self._kind = "cache"
        _LIVE.add(self)
        try:
            self._desc.k = self._malloc(n.value)
            self._desc.v = self._malloc(n.value)
        except L.HIPError:
            self.close()
            raise

    def _malloc(self, n: int) -> int:
        p = C.c_void_p()
        L.check(L.lib().ahip_malloc(self.context.handle, n, C.byref(p)))
        return p.value

    def store(self, k: int, v: int, tokens: int, start: int = 0, dtype: str = "f32", k_stride: int | None = None,
              v_stride: int | None = None, start_dev: int | None = None, stream=None) -> None:
        """Quantises rows of keys and values into positions start.. (or *start_dev..)."""
        rc = self._store(self.context.handle, self._cache, DTYPE[dtype], k,
                         self._width if k_stride is None else k_stride, v,
                         self._width if v_stride is None else v_stride, tokens, start, start_dev, stream)
        if rc:
            L.check(rc)

    def load(self, k_out: int | None, v_out: int | None, tokens: int, start: int = 0, dtype: str = "f32",
             k_stride: int | None = None, v_stride: int | None = None, stream=None) -> None:
        """The values of positions start.. as rows."""
        rc = self._load(self.context.handle, self._cache, DTYPE[dtype], start, tokens, k_out,
                        self._width if k_stride is None else k_stride, v_out,
                        self._width if v_stride is None else v_stride, stream)
        if rc:
            L.check(rc)

    def workspace_bytes(self, tokens: int, heads: int, start: int = 0, dtype: str = "f32",
                        on_device: bool = False) -> int:
        """Bytes of workspace of an attention call with these arguments (on_device: with start_dev)."""
        n = C.c_int64()
        L.check(L.lib().ahip_attention_q4_workspace(self.context.handle, self._cache, DTYPE[dtype], tokens, heads,
                                                    start, 1 if on_device else 0, C.byref(n)))
        return n.value

    def attention(self, q: int, out: int, tokens: int, heads: int, start: int = 0, dtype: str = "f32",
                  q_stride: int | None = None, out_stride: int | None = None, start_dev: int | None = None,
                  workspace: tuple | None = None, stream=None) -> None:
        """Causal attention of queries at positions start.. (or *start_dev..).

        ``workspace`` is (address, bytes), its first WORKSPACE_ZERO bytes cleared
        once; None takes the cache's own, which grows on the first call of so many
        tokens and heads to what they need at any position (an allocation: a call
        that is captured into a graph, or calls on several streams, pass theirs)."""
        if workspace is None:
            if (tokens, heads, dtype) not in self._reserved:
                self._reserve(tokens, heads, dtype)
            work, work_bytes = self._work, self._work_bytes
        else:
            work, work_bytes = workspace
        w = heads * self.head_dim
        rc = self._attention(self.context.handle, self._cache, DTYPE[dtype], q, w if q_stride is None else q_stride,
                             tokens, heads, start, start_dev, out, w if out_stride is None else out_stride, work,
                             work_bytes, stream)
        if rc:
            L.check(rc)

    def _reserve(self, tokens: int, heads: int, dtype: str) -> None:
        # the need grows with the positions seen, so the capacity's serves all
        need = self.workspace_bytes(tokens, heads, 0, dtype, True)
        if need > self._work_bytes:
            if self._work:
                # hipFree waits for the device: queued calls may still use the old one
                L.check(L.lib().ahip_free(self.context.handle, self._work))
                self._work, self._work_bytes = None, 0
                self._reserved.clear()  # (none has one should the next fail)
            self._work = self._malloc(need)
            L.check(L.lib().ahip_memset(self.context.handle, self._work, 0, WORKSPACE_ZERO))
            self._work_bytes = need
        self._reserved.add((tokens, heads, dtype))

    def close(self) -> None:
        """Frees the cache (as its context's close does); calls on it are refused."""
        for p in (self._desc.k, self._desc.v, self._work):
            if p and getattr(self.context, "handle", None):
                L.lib().ahip_free(self.context.handle, p)
        self._desc.k = self._desc.v = self._work = None
        self._work_bytes = 0
        self._reserved.clear()

    def __del__(self):
        if hasattr(self, "_desc"):
            self.close()


class PagedBatch:
    """A step of many sequences (``ahip_paged_batch``): device addresses of int32 ``row_starts`` [sequences + 1],
    ``lengths`` [sequences] (the new tokens included) and ``table`` [sequences][table_stride], which the kernels
    read; ``rows`` in all, and at most ``max_rows`` of a sequence (0: not known)."""

    def __init__(self, row_starts: int, lengths: int, table: int, sequences: int, table_stride: int, rows: int,
                 max_rows: int = 0):
        self._desc = L.PagedBatchC(row_starts, lengths, table, sequences, table_stride, rows, max_rows)
        self._ref = C.byref(self._desc)


class PagedCache:
    """Keys and values in f16, in ``pages`` pages of ``page_tokens`` tokens."""

    def __init__(self, context: HIPContext, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64):
        lib, n = L.lib(), C.c_int64()
        L.check(lib.ahip_paged_kv_bytes(kv_heads, head_dim, page_tokens, pages, C.byref(n)))
        self.context, self.pages, self.kv_heads = context, pages, kv_heads
        self.head_dim, self.page_tokens, self.bytes = head_dim, page_tokens, 2 * n.value
        self._desc = L.PagedKVC(None, None, kv_heads, head_dim, page_tokens, pages)
        self._cache = C.byref(self._desc)
        self._width = kv_heads * head_dim
        self._append, self._load, self._attention = lib.ahip_paged_append, lib.ahip_paged_load, lib.ahip_paged_attention
        self._work, self._work_bytes = None, 0
        self._kind = "cache"
        _LIVE.add(self)
        try:
            self._desc.k = self._malloc(n.value)
            self._desc.v = self._malloc(n.value)
        except L.HIPError:
            self.close()
            raise

    def _malloc(self, n: int) -> int:
        p = C.c_void_p()
        L.check(L.lib().ahip_malloc(self.context.handle, n, C.byref(p)))
        return p.value

    def append(self, batch: PagedBatch, k: int, v: int, q: int | None = None, q_out: int | None = None, heads: int = 0,
               dtype: str = "f32", rope: int | None = None, rope_positions: int = 0, interleaved: bool = True,
               q_stride: int | None = None, k_stride: int | None = None, v_stride: int | None = None,
               q_out_stride: int | None = None, stream=None) -> None:
        """Writes the batch's keys (rotated, where a table is given) and values, and its rotated queries to q_out."""
        w, qw = self._width, heads * self.head_dim
        args = _PAGED_ROWS(q or 0, q_out or 0, k or 0, v or 0, qw if q_stride is None else q_stride,
                           qw if q_out_stride is None else q_out_stride, w if k_stride is None else k_stride,
                           w if v_stride is None else v_stride, rope or 0, rope_positions, 1 if interleaved else 0,
                           DTYPE[dtype], heads)
        rc = self._append(self.context.handle, self._cache, batch._ref, args, stream)
        if rc:
            L.check(rc)

    def load(self, batch: PagedBatch, k_out: int | None, v_out: int | None, dtype: str = "f32",
             k_stride: int | None = None, v_stride: int | None = None, stream=None) -> None:
        """The cache's values at the positions of the batch's rows, as rows."""
        rc = self._load(self.context.handle, self._cache, batch._ref, DTYPE[dtype], k_out,
                        self._width if k_stride is None else k_stride, v_out,
                        self._width if v_stride is None else v_stride, stream)
        if rc:
            L.check(rc)

    def workspace_bytes(self) -> int:
        """Bytes of workspace of any attention call on this cache."""
        n = C.c_int64()
        L.check(L.lib().ahip_paged_attention_workspace(self._cache, C.byref(n)))
        return n.value

    def attention(self, batch: PagedBatch, q: int, out: int, heads: int, dtype: str = "f32", window: int = 0,
                  sinks: int = 0, q_stride: int | None = None, out_stride: int | None = None,
                  workspace: tuple | None = None, stream=None) -> None:
        """Causal attention of the batch's queries, over all positions or the last ``window`` and first ``sinks``.

        ``workspace`` is (address, bytes), its first PAGED_WORKSPACE_ZERO bytes cleared once; None takes the
        cache's own, allocated by the first such call (so a call that is captured into a graph, or calls on several
        streams, pass theirs)."""
        if workspace is None:
            if self._work is None:
                self._reserve()
            work, work_bytes = self._work, self._work_bytes
        else:
            work, work_bytes = workspace
        w = heads * self.head_dim
        rc = self._attention(self.context.handle, self._cache, batch._ref, DTYPE[dtype], q,
                             w if q_stride is None else q_stride, heads, window, sinks, out,
                             w if out_stride is None else out_stride, work, work_bytes, stream)
        if rc:
            L.check(rc)

    def _reserve(self) -> None:
        need = self.workspace_bytes()
        work = self._malloc(need)
        self._work, self._work_bytes = work, need
        try:
            L.check(L.lib().ahip_memset(self.context.handle, work, 0, PAGED_WORKSPACE_ZERO))
        except L.HIPError:
            L.lib().ahip_free(self.context.handle, work)
            self._work, self._work_bytes = None, 0
            raise

    def close(self) -> None:
        """Frees the cache (as its context's close does); calls on it are refused."""
        for p in (self._desc.k, self._desc.v, self._work):
            if p and getattr(self.context, "handle", None):
                L.lib().ahip_free(self.context.handle, p)
        self._desc.k = self._desc.v = self._work = None
        self._work_bytes = 0

    def __del__(self):
        if hasattr(self, "_desc"):
            self.close()


def rope_table(positions: int, head_dim: int, theta: float) -> np.ndarray:
    """(cos, sin) of every position and pair, [positions, head_dim / 2, 2] float32 on the host."""
    t = np.empty((positions, head_dim // 2, 2), np.float32)
    L.check(L.lib().ahip_rope_table(positions, head_dim, theta, t.ctypes.data))
    return t


def qk_norm_rope(context: HIPContext, q: int | None, k: int | None, tokens: int, heads: int, kv_heads: int,
                 head_dim: int, q_out: int | None, k_out: int | None, dtype: str = "f32", q_gain: int | None = None,
                 k_gain: int | None = None, eps: float = 1e-5, rope: int | None = None, rope_positions: int = 0,
                 interleaved: bool = True, start: int = 0, positions: int | None = None, q_stride: int | None = None,
                 k_stride: int | None = None, q_out_stride: int | None = None, k_out_stride: int | None = None,
                 stream=None) -> None:
    """Per-head RMS norm of queries and keys (where a gain is given) and their
    rotation (where a table is), ahip_qk_norm_rope."""
    qw, kw = heads * head_dim, kv_heads * head_dim
    args = _NORM_ROPE(q or 0, q_out or 0, q_gain or 0, qw if q_stride is None else q_stride,
                      qw if q_out_stride is None else q_out_stride, k or 0, k_out or 0, k_gain or 0,
                      kw if k_stride is None else k_stride, kw if k_out_stride is None else k_out_stride, rope or 0,
                      positions or 0, DTYPE[dtype], tokens, heads, kv_heads, head_dim, rope_positions,
                      1 if interleaved else 0, start, eps)
    rc = L.lib().ahip_qk_norm_rope(context.handle, args, stream)
    if rc:
        L.check(rc)
