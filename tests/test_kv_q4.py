"""What the entry points of the 4-bit KV cache refuse, and their size
arithmetic: checked before any device call, so on the CPU."""
import ctypes as C

import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd.kvcache import rope_table
from tests import q4_reference as ref

# Stands for a context (device 0, null stream) in calls that are refused before they use it.
CTX = C.create_string_buffer(64)
ctx = C.addressof(CTX)
P = 1 << 20  # a pointer that no refused call follows, 16-byte aligned
F32, F16 = L.F32, L.F16


def refused(rc, what, code=L.INVALID_ARGUMENT):
    assert rc == code
    assert what.encode() in L.lib().ahip_last_error(), L.lib().ahip_last_error()


def test_cache_bytes():
    n = C.c_int64()
    for kv_heads, cap, hd in ((1, 1, 32), (3, 8192, 64), (8, 33, 128), (5, 131072, 256)):
        assert L.lib().ahip_kv_q4_bytes(kv_heads, cap, hd, C.byref(n)) == 0
        assert n.value == kv_heads * -(-cap // 32) * 32 * hd // 32 * 18  # 18 bytes for 32 values, whole tiles
    # past 32 bits
    assert L.lib().ahip_kv_q4_bytes(8, 1 << 24, 128, C.byref(n)) == 0 and n.value == 8 * (1 << 24) * 72
    for bad in ((0, 1, 64), (1, 0, 64), (1, 1, 0), (1, 1, 48), (1, 1, 288), (-1, 1, 64), (1, -5, 64), (70000, 1, 64)):
        assert L.lib().ahip_kv_q4_bytes(*bad, C.byref(n)) == L.INVALID_ARGUMENT
    refused(L.lib().ahip_kv_q4_bytes(1, 1, 64, None), "null")


def cache(kc=P, vc=P, kv_heads=2, hd=64, cap=100):
    return C.byref(L.KVQ4C(kc, vc, kv_heads, hd, cap))


def store(ctx=ctx, dtype=F32, k=P, ks=128, v=P, vs=128, tokens=4, start=0, start_dev=None, **c):
    return L.lib().ahip_kv_q4_store(ctx, cache(**c), dtype, k, ks, v, vs, tokens, start, start_dev, None)


def test_store_refusals():
    refused(store(ctx=None), "null context")
    for dtype in (L.Q8_0, L.Q4_0, -1, 9):
        refused(store(dtype=dtype), "rows must be")
    refused(store(kc=None), "null cache")
    refused(store(vc=P + 8), "aligned")
    refused(store(hd=48), "head dimension")
    refused(store(kv_heads=0), "cache shape")
    refused(store(cap=0), "cache shape")
    refused(store(k=None), "null keys")
    refused(store(v=P + 2), "values: misaligned")
    refused(store(dtype=F16, v=P + 1), "values: misaligned")
    refused(store(ks=127), "keys: stride")
    refused(store(vs=-1), "values: stride")
    refused(store(start=97), "capacity")
    refused(store(start=-1), "capacity")
    refused(store(start=2**31 - 1), "capacity")
    refused(store(tokens=101), "more tokens")
    refused(store(tokens=-1), "more tokens")
    refused(store(tokens=101, start_dev=P), "more tokens")
    refused(store(start_dev=P + 1), "start_dev")
    assert store(tokens=0, k=None, v=None) == 0  # nothing to do


def load(ctx=ctx, dtype=F32, start=0, tokens=4, k=P, ks=128, v=P, vs=128, **c):
    return L.lib().ahip_kv_q4_load(ctx, cache(**c), dtype, start, tokens, k, ks, v, vs, None)


def test_load_refusals():
    refused(load(ctx=None), "null context")
    refused(load(dtype=L.Q4_0), "rows must be")
    refused(load(kc=None), "null cache")
    refused(load(start=98), "capacity")
    refused(load(tokens=101), "more tokens")
    refused(load(k=P + 2), "keys: misaligned")
    refused(load(vs=100), "values: stride")
    assert load(tokens=0) == 0 and load(k=None, v=None) == 0


def attention(ctx=ctx, dtype=F32, q=P, qs=256, tokens=4, heads=4, start=10, start_dev=None, out=P, os=256, ws=None,
              wb=0, **c):
    return L.lib().ahip_attention_q4(ctx, cache(**c), dtype, q, qs, tokens, heads, start, start_dev, out, os, ws, wb,
                                     None)


def test_attention_refusals():
    refused(attention(ctx=None), "null context")
    refused(attention(dtype=L.Q8_0), "rows must be")
    refused(attention(kc=None), "null cache")
    refused(attention(vc=P + 4), "aligned")
    refused(attention(heads=5), "multiple of the KV heads")
    refused(attention(heads=0), "multiple of the KV heads")
    refused(attention(kv_heads=0), "cache shape")
    refused(attention(hd=80), "head dimension")
    refused(attention(start=97), "capacity")
    refused(attention(start=-1), "capacity")
    refused(attention(tokens=101), "more tokens")
    refused(attention(tokens=-1), "more tokens")
    refused(attention(start_dev=P + 2), "start_dev")
    refused(attention(q=None), "null queries")
    refused(attention(out=None), "null output")
    refused(attention(qs=255), "queries: stride")
    refused(attention(os=255), "output: stride")
    refused(attention(q=P + 2), "queries: misaligned")
    refused(attention(tokens=1 << 20, heads=4096, kv_heads=4096, cap=1 << 30), "2^30", L.UNSUPPORTED)
    assert attention(tokens=0, q=None, out=None) == 0


def test_workspace_refusals():
    n = C.c_int64()

    def f(ctx=ctx, dtype=F32, tokens=1, heads=4, start=0, on_device=0, n=n, **c):
        return L.lib().ahip_attention_q4_workspace(ctx, cache(**c), dtype, tokens, heads, start, on_device,
                                                   None if n is None else C.byref(n))
    refused(f(ctx=None), "null")
    refused(f(n=None), "null")
    refused(f(dtype=L.Q4_0), "rows must be")
    refused(f(heads=5), "multiple")
    refused(f(hd=65), "head dimension")
    refused(f(start=100), "capacity")
    refused(f(tokens=101, on_device=1), "more tokens")
    refused(L.lib().ahip_attention_q4_workspace(ctx, None, F32, 1, 4, 0, 0, C.byref(n)), "null cache")
    n.value = 7
    assert f(tokens=0) == 0 and n.value == 0


def norm_rope(ctx=ctx, dtype=F32, q=P, qs=256, heads=4, qg=P, k=P, ks=128, kv_heads=2, kg=P, tokens=4, hd=64, eps=1e-5,
              rope=P, positions=100, start=0, pos=None, qo=P, qos=256, ko=P, kos=128):
    a = L.NormRopeC(q, qo, qg, qs, qos, k, ko, kg, ks, kos, rope, pos, dtype, tokens, heads, kv_heads, hd, positions,
                    1, start, eps)
    return L.lib().ahip_qk_norm_rope(ctx, C.byref(a), None)


def test_norm_rope_refusals():
    refused(norm_rope(ctx=None), "null context")
    refused(L.lib().ahip_qk_norm_rope(ctx, None, None), "null arguments")
    refused(norm_rope(dtype=L.Q8_0), "rows must be")
    refused(norm_rope(hd=72), "head dimension")
    refused(norm_rope(heads=-1), "head counts")
    refused(norm_rope(tokens=-1), "token count")
    refused(norm_rope(eps=-1.0), "eps")
    refused(norm_rope(eps=float("nan")), "eps")
    refused(norm_rope(qg=P + 1), "gain")
    refused(norm_rope(rope=P + 4), "rotation table")
    refused(norm_rope(positions=0), "rotation table")
    refused(norm_rope(start=97), "rotation table")
    refused(norm_rope(start=-1), "rotation table")
    refused(norm_rope(start=2**31 - 1), "rotation table")
    refused(norm_rope(pos=P + 2), "positions")
    refused(norm_rope(q=None), "null queries")
    refused(norm_rope(qo=None), "null query output")
    refused(norm_rope(ks=100), "keys: stride")
    refused(norm_rope(kos=127), "key output: stride")
    refused(norm_rope(ko=P + 2), "key output: misaligned")
    refused(norm_rope(tokens=1 << 29, rope=None), "2^30", L.UNSUPPORTED)
    assert norm_rope(tokens=0, q=None, k=None, qo=None, ko=None) == 0
    assert norm_rope(heads=0, kv_heads=0) == 0


def test_rotation_table_is_the_double_angle_rounded_once():
    t = rope_table(300, 96, 1e5)
    a = np.arange(300)[:, None] * 1e5 ** (-2.0 * np.arange(48) / 96)
    np.testing.assert_allclose(t[..., 0], np.cos(a), rtol=0, atol=6.1e-8)
    np.testing.assert_allclose(t[..., 1], np.sin(a), rtol=0, atol=6.1e-8)
    with pytest.raises(L.InvalidArgument):
        rope_table(4, 64, 0.0)
    for bad in ((-1, 64), (4, 0), (4, 63), (1, 1 << 20)):  # (refused before the table is written)
        refused(L.lib().ahip_rope_table(*bad, 1e4, None if bad[0] < 0 else P), "rotation table")
    assert rope_table(0, 64, 1e4).shape == (0, 32, 2)


def test_the_reference_reads_back_what_the_quantiser_writes():
    from alpaca_amd.tensor import Q4_0, quantize
    import oracle.oracle as orc
    x = (np.random.default_rng(2).standard_normal((50, 3, 64)) * 3).astype(np.float32)
    want = orc.dequantize(orc.Q4_0, quantize(x, Q4_0), x.size).reshape(x.shape)
    assert np.array_equal(ref.q4_values(x), want.astype(np.float64))


def test_the_packed_arguments_are_the_structure_s_bytes():
    from alpaca_amd import kvcache
    values = [P + 64 * i for i in range(3)] + [7, 8] + [P + 4096 + 64 * i for i in range(3)] + [9, 10, P + 16, P + 32, 1,
                                                                                        2, 3, 4, 64, 5, 1, 6, 1e-5]
    assert kvcache._NORM_ROPE(*values) == bytes(L.NormRopeC(*values))
