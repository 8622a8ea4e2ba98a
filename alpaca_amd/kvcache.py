"""A KV cache held in 4 bits on the device, and the operators around it.

``Q4Cache`` owns one layer's cache (``ahip_kv_q4_*``, ``ahip_attention_q4`` of
include/alpaca_hip.h) and the attention's workspace; ``qk_norm_rope`` is the
per-head norm of queries and keys with their rotation.  Rows, outputs, gains
and tables are device addresses (``ahip_malloc``, or any allocator of the same
device), rows [tokens][heads][head_dim] of ``dtype`` "f32" or "f16" with
``stride`` elements from one token to the next (None: dense).  Work is queued on
``stream`` (a handle of ``ahip_stream_create``; None: the context's stream), in
order and without waiting.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib as L
from .model import HIPContext, _LIVE

DTYPE = {"f32": L.F32, "f16": L.F16}


class Q4Cache:
    """Keys and values of up to ``capacity`` tokens, Q4_0 blocks along the head dimension."""

    def __init__(self, context: HIPContext, kv_heads: int, capacity: int, head_dim: int):
        n = C.c_int64()
        L.check(L.lib().ahip_kv_q4_bytes(kv_heads, capacity, head_dim, C.byref(n)))
        self.context, self.kv_heads, self.capacity, self.head_dim = context, kv_heads, capacity, head_dim
        self.bytes = 2 * n.value
        self._k = self._v = self._work = None
        self._work_bytes = 0
        self._needs = {}
        self._kind = "cache"
        _LIVE.add(self)
        self._k, self._v = self._malloc(n.value), self._malloc(n.value)

    def _malloc(self, n: int) -> int:
        p = C.c_void_p()
        L.check(L.lib().ahip_malloc(self.context.handle, n, C.byref(p)))
        return p.value

    def store(self, k: int, v: int, tokens: int, start: int = 0, dtype: str = "f32", k_stride: int | None = None,
              v_stride: int | None = None, start_dev: int | None = None, stream=None) -> None:
        """Quantises rows of keys and values into positions start.. (or *start_dev..)."""
        w = self.kv_heads * self.head_dim
        L.check(L.lib().ahip_kv_q4_store(self.context.handle, DTYPE[dtype], k, w if k_stride is None else k_stride, v,
                                         w if v_stride is None else v_stride, tokens, start, start_dev, self._k,
                                         self._v, self.kv_heads, self.head_dim, self.capacity, stream))

    def load(self, k_out: int | None, v_out: int | None, tokens: int, start: int = 0, dtype: str = "f32",
             k_stride: int | None = None, v_stride: int | None = None, stream=None) -> None:
        """The values of positions start.. as rows."""
        w = self.kv_heads * self.head_dim
        L.check(L.lib().ahip_kv_q4_load(self.context.handle, DTYPE[dtype], self._k, self._v, self.kv_heads,
                                        self.head_dim, self.capacity, start, tokens, k_out,
                                        w if k_stride is None else k_stride, v_out,
                                        w if v_stride is None else v_stride, stream))

    def workspace_bytes(self, tokens: int, heads: int, start: int = 0, on_device: bool = False) -> int:
        n = C.c_int64()
        L.check(L.lib().ahip_attention_q4_workspace(self.context.handle, tokens, heads, self.kv_heads, self.head_dim,
                                                    start, 1 if on_device else 0, self.capacity, C.byref(n)))
        return n.value

    def attention(self, q: int, out: int, tokens: int, heads: int, start: int = 0, dtype: str = "f32",
                  q_stride: int | None = None, out_stride: int | None = None, start_dev: int | None = None,
                  workspace: tuple | None = None, stream=None) -> None:
        """Causal attention of queries at positions start.. (or *start_dev..).

        ``workspace`` is (address, bytes); None takes the cache's own, which
        grows to what the calls so far needed (an allocation: a call that is
        captured into a graph, or calls on several streams, pass theirs)."""
        w = heads * self.head_dim
        if workspace is None:
            key = (tokens, heads, start, start_dev is not None)
            need = self._needs.get(key)
            if need is None:
                need = self._needs[key] = self.workspace_bytes(tokens, heads, start, start_dev is not None)
                if len(self._needs) > 1024:
                    self._needs = {key: need}
            if need > self._work_bytes:
                self._grow(need)
            workspace = (self._work, self._work_bytes)
        L.check(L.lib().ahip_attention_q4(self.context.handle, DTYPE[dtype], q, w if q_stride is None else q_stride,
                                          tokens, heads, start, start_dev, self._k, self._v, self.kv_heads,
                                          self.head_dim, self.capacity, out, w if out_stride is None else out_stride,
                                          workspace[0], workspace[1], stream))

    def _grow(self, need: int) -> None:
        if self._work:
            # hipFree waits for the device: queued calls may still use the old one
            L.check(L.lib().ahip_free(self.context.handle, self._work))
            self._work, self._work_bytes = None, 0
        self._work = self._malloc(need)
        self._work_bytes = need

    def close(self) -> None:
        if not getattr(self.context, "handle", None):
            return
        for p in (self._k, self._v, self._work):
            if p:
                L.lib().ahip_free(self.context.handle, p)
        self._k = self._v = self._work = None
        self._work_bytes = 0

    def __del__(self):
        if hasattr(self, "_k"):
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
    L.check(L.lib().ahip_qk_norm_rope(
        context.handle, DTYPE[dtype], q, qw if q_stride is None else q_stride, heads, q_gain, k,
        kw if k_stride is None else k_stride, kv_heads, k_gain, tokens, head_dim, eps, rope, rope_positions,
        1 if interleaved else 0, start, positions, q_out, qw if q_out_stride is None else q_out_stride, k_out,
        kw if k_out_stride is None else k_out_stride, stream))
