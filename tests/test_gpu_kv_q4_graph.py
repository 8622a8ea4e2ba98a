"""The device calls of the 4-bit KV cache captured into a HIP graph that follows
a position on the device, replayed with eager calls between."""
import ctypes as C

import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd.kvcache import Q4Cache, qk_norm_rope, rope_table
from tests import q4_reference as ref
from tests.test_gpu_kv_q4 import NP, rows, run_attention, store

pytestmark = pytest.mark.gpu


class Stream(C.Structure):  # ahip_stream
    _fields_ = [("device", C.c_int), ("handle", C.c_void_p)]


def capture(stream, calls):
    """An executable graph of what `calls` queues on `stream`, and how to launch and destroy it."""
    hip = C.CDLL("libamdhip64.so")
    handle = C.c_void_p(C.cast(stream, C.POINTER(Stream)).contents.handle)
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(handle, 1) == 0  # (thread local)
    calls()
    assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, C.c_size_t(0)) == 0
    assert hip.hipGraphDestroy(graph) == 0

    def launch():
        assert hip.hipGraphLaunch(graph_exec, handle) == 0
        L.check(L.lib().ahip_stream_synchronize(stream))
    return launch, lambda: hip.hipGraphExecDestroy(graph_exec)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,capacity", [
    (9, 3, 64, 1, 5000), (8, 2, 128, 1, 3000), (6, 2, 64, 40, 4000), (64, 64, 128, 260, 700)])
def test_a_layer_s_step_follows_its_position(hip_ctx, heads, kv_heads, hd, tokens, capacity, dtype):
    rng = np.random.default_rng(heads + hd)
    t = NP[dtype]
    size, w, wk = t().nbytes, heads * hd, kv_heads * hd
    stream = C.c_void_p()
    L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(stream)))
    table, gain = rope_table(capacity, hd, 1e5), (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    old = [rows(rng, capacity, kv_heads, hd, dtype) for _ in range(2)]
    caches = [Q4Cache(hip_ctx, kv_heads, capacity, hd) for _ in range(2)]
    with ref.Device(hip_ctx) as dev:
        for c in caches:
            for p in (c._desc.k, c._desc.v):  # (the padding behind the last position, for the comparison)
                L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0, c.bytes // 2))
            store(dev, c, *old, 0, dtype)
        tab, g = dev.put(table), dev.put(gain)
        q, k, v, qr, kr, out = (dev.empty(tokens * n * size) for n in (w, wk, wk, w, wk, w))
        start, positions = dev.empty(4), dev.empty(4 * tokens)
        need = caches[0].workspace_bytes(tokens, heads, 0, dtype, True)
        works = [(dev.empty(max(need, 16), 0), need) for _ in range(2)]

        def step(cache, work, s):
            qk_norm_rope(hip_ctx, q, k, tokens, heads, kv_heads, hd, qr, kr, dtype, g, g, 1e-6, tab, capacity,
                         positions=positions, stream=s)
            cache.store(kr, v, tokens, 0, dtype, start_dev=start, stream=s)
            cache.attention(qr, out, tokens, heads, 0, dtype, start_dev=start, workspace=work, stream=s)
        launch, destroy = capture(stream, lambda: step(caches[0], works[0], stream))

        def put(p, a):
            L.check(L.lib().ahip_memcpy_htod(hip_ctx.handle, p, np.ascontiguousarray(a).ctypes.data, a.nbytes))
        at = [0, 31, capacity - tokens, 7, capacity // 2, capacity // 2, 1]
        for i, pos in enumerate(at):
            new = rows(rng, tokens, heads, hd, dtype), *(rows(rng, tokens, kv_heads, hd, dtype) for _ in range(2))
            for p, a in zip((q, k, v), new):
                put(p, a)
            put(start, np.array([pos], np.int32))
            put(positions, pos + np.arange(tokens, dtype=np.int32))
            launch()
            got = [dev.get(p, (tokens, n, hd), t) for p, n in ((out, heads), (kr, kv_heads), (qr, heads))]
            for p, n in ((out, w), (kr, wk), (qr, w)):
                L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0xA5, tokens * n * size))
            step(caches[1], works[1], None)  # the program's own eager work, on its own cache
            want = [dev.get(p, (tokens, n, hd), t) for p, n in ((out, heads), (kr, kv_heads), (qr, heads))]
            assert np.isfinite(want[0]).all()
            assert all(np.array_equal(a, b) for a, b in zip(got, want)), (i, pos)
            # and a call of other sizes over the graph's cache, with the cache's own workspace
            run_attention(dev, caches[0], rows(rng, 3, heads, hd, dtype), capacity - 3, dtype)
        data = [dev.get(p, c.bytes // 2, np.uint8) for c in caches for p in (c._desc.k, c._desc.v)]
        assert np.array_equal(data[0], data[2]) and np.array_equal(data[1], data[3])
        assert not any(dev.get(p, min(n, 2048), np.uint8).any() for p, n in works)
        destroy()
    L.check(L.lib().ahip_stream_destroy(stream))
