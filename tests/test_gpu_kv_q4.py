"""The KV cache held in 4 bits on the GPU: writing and reading back bit for bit,
the attention over it and the norm with rotation against 64-bit plain forms."""
import numpy as np
import pytest

import oracle.oracle as orc
from alpaca_amd import _lib as L
from alpaca_amd.kvcache import WORKSPACE_ZERO, Q4Cache, qk_norm_rope, rope_table
from alpaca_amd.tensor import Q4_0
from tests import q4_reference as ref

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "f16": np.float16}


def rows(rng, tokens, heads, hd, dtype, size=1.0):
    return (rng.standard_normal((tokens, heads, hd)) * size).astype(NP[dtype])


def padded(x, extra, fill=7.0):
    """Rows with `extra` elements behind each token's, and their stride."""
    flat = x.reshape(len(x), -1)
    out = np.full((len(x), flat.shape[1] + extra), fill, x.dtype)
    out[:, :flat.shape[1]] = flat
    return out, flat.shape[1] + extra


def store(dev, cache, k, v, start, dtype, extra=(0, 0), **kw):
    (kp, ks), (vp, vs) = padded(k, extra[0]), padded(v, extra[1])
    cache.store(dev.put(kp), dev.put(vp), len(k), start, dtype, k_stride=ks, v_stride=vs, **kw)


def load(dev, cache, start, tokens, dtype, extra=0):
    w = cache.kv_heads * cache.head_dim
    ko, vo = (dev.empty(tokens * (w + extra) * NP[dtype]().nbytes) for _ in range(2))
    cache.load(ko, vo, tokens, start, dtype, k_stride=w + extra, v_stride=w + extra)
    out = []
    for p in (ko, vo):
        a = dev.get(p, (tokens, w + extra), NP[dtype])
        if extra:  # what lies between the rows stays
            assert (a[:, w:].view(np.uint8) == 0xA5).all()
        out.append(a[:, :w].reshape(tokens, cache.kv_heads, cache.head_dim))
    return out


def equal(a, b):
    """Equal values, NaN for NaN (a zero's sign is not compared)."""
    return np.array_equal(a.astype(np.float64), b.astype(np.float64), equal_nan=True)


# ---------------------------------------------------------------- store, load

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kv_heads,hd,tokens,start,capacity", [
    (3, 64, 1, 0, 1), (3, 64, 1, 31, 64), (2, 128, 32, 0, 32), (2, 128, 33, 31, 64), (1, 32, 7, 60, 67),
    (5, 96, 64, 32, 100), (2, 160, 100, 5, 200), (1, 192, 3, 62, 65), (2, 224, 40, 1, 41), (3, 256, 70, 30, 128),
    (32, 64, 257, 1000, 1300)])
def test_store_and_load_are_the_quantiser_bit_for_bit(hip_ctx, dtype, kv_heads, hd, tokens, start, capacity):
    rng = np.random.default_rng(tokens * 1000 + hd)
    k, v = rows(rng, tokens, kv_heads, hd, dtype, 4), rows(rng, tokens, kv_heads, hd, dtype, 0.02)
    cache = Q4Cache(hip_ctx, kv_heads, capacity, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, start, dtype, extra=(3, 8))
        got32, got16 = load(dev, cache, start, tokens, "f32", 5), load(dev, cache, start, tokens, "f16")
    cache.close()
    for x, g32, g16 in zip((k, v), got32, got16):
        raw = orc.quantize(x.astype(np.float32).ravel(), Q4_0)
        want = orc.dequantize(orc.Q4_0, raw, x.size).reshape(x.shape)
        assert equal(g32, want) and equal(ref.q4_values(x.astype(np.float32)), want)
        assert equal(g16, want.astype(np.float16))


def test_values_at_the_format_s_edges(hip_ctx):
    """Zero blocks, ties of the largest magnitude, one value alone, scales below f16's range, its largest value."""
    x = np.zeros((9, 1, 64), np.float32)
    x[1, 0, :32] = -2.5                                 # all equal
    x[2, 0, 3], x[2, 0, 40] = 1e-30, -1e-42             # scales that f16 rounds to zero
    x[3, 0, 5], x[3, 0, 6] = 3, -3                      # a tie: the first one sets the scale's sign
    x[3, 0, 36], x[3, 0, 35] = 3, -3
    x[4, 0, 31], x[4, 0, 0] = 65504, -65504
    x[5, 0] = np.linspace(-1, 1, 64)
    x[6, 0, :32] = np.float32(2.0 ** -24) * np.arange(32)  # a scale in f16's subnormals
    x[7, 0, 1::2] = -0.0
    x[8, 0] = np.arange(64) * 8 + 4                     # values on the borders of a step
    cache = Q4Cache(hip_ctx, 1, 40, 64)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, x, -x, 30, "f32")
        k, v = load(dev, cache, 30, 9, "f32")
    assert equal(k, ref.q4_values(x)) and equal(v, ref.q4_values(-x))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 70000.0])
def test_a_token_without_a_form_is_nan_in_its_head_only(hip_ctx, dtype, value):
    rng = np.random.default_rng(3)
    k, v = rows(rng, 40, 2, 64, dtype), rows(rng, 40, 2, 64, dtype)
    with np.errstate(over="ignore"):
        k[7, 1, 63], v[20, 0, 0] = value, value
    cache = Q4Cache(hip_ctx, 2, 40, 64)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, dtype)
        got = load(dev, cache, 0, 40, "f32")
    want = ref.q4_rows(k.astype(np.float32), v.astype(np.float32))
    assert np.isnan(want[0]).sum() == np.isnan(want[1]).sum() == 2 * 64
    assert all(equal(g, w) for g, w in zip(got, want))


def test_positions_that_are_not_written_keep_their_bytes(hip_ctx):
    rng = np.random.default_rng(4)
    k, v = rows(rng, 100, 3, 96, "f32"), rows(rng, 100, 3, 96, "f32")
    want = [ref.q4_values(x) for x in (k, v)]
    cache = Q4Cache(hip_ctx, 3, 100, 96)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        before = [dev.get(p, cache.bytes // 2, np.uint8) for p in (cache._desc.k, cache._desc.v)]
        for start, n in ((37, 1), (50, 20), (0, 2), (99, 1), (64, 32)):
            a, b = rows(rng, n, 3, 96, "f32"), rows(rng, n, 3, 96, "f32")
            store(dev, cache, a, b, start, "f32")
            want[0][start:start + n], want[1][start:start + n] = ref.q4_values(a), ref.q4_values(b)
            got = load(dev, cache, 0, 100, "f32")
            assert all(equal(g, w) for g, w in zip(got, want)), (start, n)
        # the padding behind the last position is never written
        cache.store(dev.put(k), dev.put(v), 100, 0)
        after = [dev.get(p, cache.bytes // 2, np.uint8) for p in (cache._desc.k, cache._desc.v)]
    assert all(np.array_equal(a, b) for a, b in zip(before, after))


def test_store_at_a_position_on_the_device(hip_ctx):
    rng = np.random.default_rng(5)
    cache = Q4Cache(hip_ctx, 2, 80, 64)
    base = rows(rng, 80, 2, 64, "f32"), rows(rng, 80, 2, 64, "f32")
    want = [ref.q4_values(x) for x in base]
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, *base, 0, "f32")
        for n, start in ((1, 0), (1, 79), (33, 31), (34, 46), (2, 79), (1, 80), (5, -1), (80, 0), (80, 1)):
            k, v = rows(rng, n, 2, 64, "f32"), rows(rng, n, 2, 64, "f32")
            store(dev, cache, k, v, 0, "f32", start_dev=dev.put(np.array([start], np.int32)))
            if 0 <= start <= 80 - n:  # a range outside the cache writes nothing
                want[0][start:start + n], want[1][start:start + n] = ref.q4_values(k), ref.q4_values(v)
            got = load(dev, cache, 0, 80, "f32")
            assert all(equal(g, w) for g, w in zip(got, want)), (n, start)


def test_load_of_one_of_the_two(hip_ctx):
    rng = np.random.default_rng(6)
    k, v = rows(rng, 50, 1, 32, "f32"), rows(rng, 50, 1, 32, "f32")
    cache = Q4Cache(hip_ctx, 1, 50, 32)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        p = dev.empty(50 * 32 * 4)
        cache.load(None, p, 50)
        assert equal(dev.get(p, (50, 1, 32), np.float32), ref.q4_values(v))
        cache.load(p, None, 50)
        assert equal(dev.get(p, (50, 1, 32), np.float32), ref.q4_values(k))


# ---------------------------------------------------------------- attention

def run_attention(dev, cache, q, start, dtype, extra=0, **kw):
    T, H, hd = q.shape
    qp, qs = padded(q, extra)
    out = dev.empty(T * (H * hd + extra) * q.itemsize)
    cache.attention(dev.put(qp), out, T, H, start, dtype, q_stride=qs, out_stride=H * hd + extra, **kw)
    a = dev.get(out, (T, H * hd + extra), q.dtype)
    if extra:
        assert (a[:, H * hd:].view(np.uint8) == 0xA5).all()
    return a[:, :H * hd].reshape(T, H, hd)


def check_attention(got, q, k, v, start, dtype, label):
    want, bound = ref.attention(q, k, v, start, dtype)
    off = np.abs(got.astype(np.float64) - want)
    near = bool((off <= bound).all())  # (a NaN is not)
    print(f"[attention] {label}: {np.max(off / np.maximum(bound, 1e-300)):.3f} of the bound, max |d| {off.max():.3e}")
    assert near, label


def attention_case(hip_ctx, heads, kv_heads, hd, tokens, start, dtype, spare=0, extra=0, q_size=3.0):
    rng = np.random.default_rng(heads * 7919 + hd * 31 + tokens * 17 + start)
    n = start + tokens
    k, v = rows(rng, n, kv_heads, hd, "f32"), rows(rng, n, kv_heads, hd, "f32")
    k *= 1 + 5 * (rng.random((kv_heads, hd)) < 0.05)
    q = rows(rng, tokens, heads, hd, dtype, q_size)
    cache = Q4Cache(hip_ctx, kv_heads, n + spare, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, start, dtype, extra)
    cache.close()
    check_attention(got, q, *ref.q4_rows(k, v), start, dtype, (heads, kv_heads, hd, tokens, start, dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("tokens,start", [(1, 0), (1, 100), (5, 30), (37, 65)])
def test_attention_at_every_head_dim(hip_ctx, hd, tokens, start, dtype):
    attention_case(hip_ctx, 6, 2, hd, tokens, start, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (4, 4), (16, 1), (17, 1), (14, 2), (40, 1), (40, 8)])
@pytest.mark.parametrize("tokens,start", [(1, 31), (1, 700), (3, 0), (18, 33)])
def test_attention_at_groups_of_query_heads(hip_ctx, heads, kv_heads, tokens, start, dtype):
    attention_case(hip_ctx, heads, kv_heads, 64, tokens, start, dtype, spare=9, extra=8)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("tokens,start", [(1, 1), (1, 32), (1, 63), (1, 64), (2, 31), (16, 0), (17, 15), (33, 0),
                                          (64, 0), (65, 64), (129, 7), (200, 1), (300, 500)])
def test_attention_around_tile_edges(hip_ctx, tokens, start, dtype):
    attention_case(hip_ctx, 4, 2, 128, tokens, start, dtype, spare=50)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", [
    (9, 3, 64, 1, 8000), (32, 8, 128, 1, 4095), (2, 1, 64, 1, 40000), (9, 3, 64, 11, 3000), (4, 1, 96, 40, 5000)])
def test_attention_over_long_caches(hip_ctx, heads, kv_heads, hd, tokens, start, dtype):
    attention_case(hip_ctx, heads, kv_heads, hd, tokens, start, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-6, 1, 1), (60, 4, 1), (1, 1, 1e-4), (1, 1e-4, 3000), (1, 300, 1),
                                                  (0, 1, 1)])
def test_attention_of_small_and_large_values(hip_ctx, q_size, k_size, v_size, dtype):
    """Near-uniform and one-hot softmaxes, scales near both ends of f16."""
    rng = np.random.default_rng(11)
    q = rows(rng, 3, 6, 64, dtype, q_size)
    k, v = rows(rng, 203, 2, 64, "f32", k_size), rows(rng, 203, 2, 64, "f32", v_size)
    cache = Q4Cache(hip_ctx, 2, 203, 64)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, 200, dtype)
    check_attention(got, q, *ref.q4_rows(k, v), 200, dtype, (q_size, k_size, v_size, dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("tokens", [1, 5, 100])
def test_a_token_without_a_form_reaches_only_the_queries_that_see_it(hip_ctx, where, tokens, dtype):
    rng = np.random.default_rng(12)
    start, n = 60, 60 + tokens
    k, v = rows(rng, n, 2, 64, "f32"), rows(rng, n, 2, 64, "f32")
    q = rows(rng, tokens, 4, 64, dtype)
    hit = start + tokens // 2
    (k if where == "k" else v)[hit, 1, 5] = np.inf
    cache = Q4Cache(hip_ctx, 2, n, 64)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, start, dtype)
    bad = np.zeros(got.shape, bool)
    bad[hit - start:, 2:] = True  # the queries of KV head 1 at and past the token
    assert np.array_equal(np.isnan(got), bad)
    (k if where == "k" else v)[hit, 1, 5] = 0
    clean = ref.q4_rows(k, v)
    want, bound = ref.attention(q, *clean, start, dtype)
    assert (np.abs(got.astype(np.float64) - want) <= bound)[~bad].all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_never_reads_positions_past_its_own(hip_ctx, dtype):
    """Rows behind the last token, of an earlier text or never written, change no bit."""
    rng = np.random.default_rng(13)
    k, v = rows(rng, 300, 2, 64, "f32"), rows(rng, 300, 2, 64, "f32")
    q = rows(rng, 20, 6, 64, dtype)
    got = []
    for tail in (0, 1, np.nan):
        cache = Q4Cache(hip_ctx, 2, 300, 64)
        with ref.Device(hip_ctx) as dev:
            for p in (cache._desc.k, cache._desc.v):
                L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0xFF, cache.bytes // 2))
            if tail != 0:
                store(dev, cache, k * tail, v * tail, 0, "f32")
            store(dev, cache, k[:90], v[:90], 0, "f32")
            got.append(run_attention(dev, cache, q, 70, dtype))
    check_attention(got[0], q, *ref.q4_rows(k[:90], v[:90]), 70, dtype, "tails")
    assert all(np.array_equal(g.view(np.uint8), got[0].view(np.uint8)) for g in got[1:])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_at_a_position_on_the_device(hip_ctx, dtype):
    rng = np.random.default_rng(14)
    cap = 1500
    k, v = rows(rng, cap, 3, 64, "f32"), rows(rng, cap, 3, 64, "f32")
    kd, vd = ref.q4_rows(k, v)
    cache = Q4Cache(hip_ctx, 3, cap, 64)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        for T, start in ((1, 0), (1, 31), (1, 1000), (1, cap - 1), (4, 500), (20, cap - 20)):
            q = rows(rng, T, 9, 64, dtype, 3)
            got = run_attention(dev, cache, q, 0, dtype, start_dev=dev.put(np.array([start], np.int32)))
            check_attention(got, q, kd[:start + T], vd[:start + T], start, dtype, ("device", T, start))
        for T, start in ((1, cap), (1, -1), (20, cap - 19)):
            q = rows(rng, T, 9, 64, dtype)
            got = run_attention(dev, cache, q, 0, dtype, start_dev=dev.put(np.array([start], np.int32)))
            assert np.isnan(got).all()


def test_attention_twice_gives_the_same_bits(hip_ctx):
    rng = np.random.default_rng(15)
    k, v = rows(rng, 3000, 2, 128, "f32"), rows(rng, 3000, 2, 128, "f32")
    q = rows(rng, 3, 8, 128, "f32")
    cache = Q4Cache(hip_ctx, 2, 3000, 128)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        a = run_attention(dev, cache, q, 2997, "f32")
        need = cache.workspace_bytes(3, 8, 2997)
        assert need > WORKSPACE_ZERO  # (the keys are split over workgroups)
        mine = (dev.empty(need, 0xFF), need)  # another workspace, its bytes NaN but for the counters
        L.check(L.lib().ahip_memset(hip_ctx.handle, mine[0], 0, WORKSPACE_ZERO))
        b = run_attention(dev, cache, q, 2997, "f32", workspace=mine)
        with pytest.raises(L.InvalidArgument, match="workspace"):
            run_attention(dev, cache, q, 2997, "f32", workspace=(mine[0], need - 1))
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def check_heads(got, q, kd, vd, start, dtype, heads, label):
    """As check_attention, for some of the query heads."""
    G = q.shape[1] // kd.shape[1]
    for h in heads:
        one, kv = slice(h, h + 1), slice(h // G, h // G + 1)
        check_attention(got[:, one], q[:, one], kd[:, kv], vd[:, kv], start, dtype, (*label, h))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", [
    (128, 128, 128, 250, 37),  # a chip full of workgroups of 128 columns
    (64, 64, 160, 250, 3), (64, 64, 192, 197, 60), (70, 70, 128, 129, 0), (64, 64, 256, 250, 0), (96, 32, 64, 350, 31),
    (300, 300, 64, 128, 21), (256, 256, 96, 150, 33), (400, 200, 32, 90, 5),  # and 32 of float32
    (130, 130, 64, 70, 1600),  # four sets of waves in f16
    (200, 200, 128, 250, 700), (180, 180, 160, 130, 300), (340, 340, 64, 129, 200),  # and one
    (600, 600, 32, 1, 2100), (16, 1, 32, 1, 5000), (8, 1, 128, 1, 5000)])
def test_attention_of_many_heads(hip_ctx, heads, kv_heads, hd, tokens, start, dtype):
    """Calls that fill the chip, at every width of a workgroup; many KV heads and long caches for few queries."""
    rng = np.random.default_rng(heads + hd)
    n = start + tokens
    k, v = rows(rng, n, kv_heads, hd, "f32"), rows(rng, n, kv_heads, hd, "f32")
    q = rows(rng, tokens, heads, hd, dtype, 3)
    cache = Q4Cache(hip_ctx, kv_heads, n + 13, hd)
    with ref.Device(hip_ctx) as dev:
        for p in (cache._desc.k, cache._desc.v):  # what was never written is NaN
            L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0xFF, cache.bytes // 2))
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, start, dtype)
        on_device = run_attention(dev, cache, q, 0, dtype, start_dev=dev.put(np.array([start], np.int32)))
    cache.close()
    kd, vd = ref.q4_rows(k, v)
    for x in (got, on_device):
        check_heads(x, q, kd, vd, start, dtype, [0, heads // 2, heads - 1], (hd, tokens))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [128, 160])
def test_a_token_without_a_form_in_a_long_prompt(hip_ctx, hd, dtype):
    rng = np.random.default_rng(16)
    H, T, hit = 64, 250, 131
    k, v = rows(rng, T, H, hd, "f32"), rows(rng, T, H, hd, "f32")
    q = rows(rng, T, H, hd, dtype)
    clean = ref.q4_rows(k, v)
    v[hit, 5, 9] = np.nan
    cache = Q4Cache(hip_ctx, H, T, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, 0, dtype)
    bad = np.zeros(got.shape, bool)
    bad[hit:, 5] = True
    assert np.array_equal(np.isnan(got), bad)
    check_heads(got[:hit], q[:hit], *[x[:hit] for x in clean], 0, dtype, [5], (hd, "before"))
    check_heads(got, q, *clean, 0, dtype, [4, 6], (hd, "beside"))


def test_one_workspace_serves_calls_of_every_shape_in_turn(hip_ctx):
    """Joined in one launch or in two, or not split: each leaves the workspace as the next needs it."""
    rng = np.random.default_rng(17)
    n = 6000
    k, v = rows(rng, n, 2, 64, "f32"), rows(rng, n, 2, 64, "f32")
    cache = Q4Cache(hip_ctx, 2, n, 64)
    shapes = [(1, 8, 5999), (64, 8, 5900), (1, 2, 200), (3, 4, 4000), (700, 8, 5300), (1, 32, 2000), (1, 8, 5999)] * 2
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        need = max(cache.workspace_bytes(T, H, at) for T, H, at in shapes)
        one = dev.empty(need)
        L.check(L.lib().ahip_memset(hip_ctx.handle, one, 0, WORKSPACE_ZERO))
        for T, H, at in shapes:
            q = rows(rng, T, H, 64, "f32")
            a = run_attention(dev, cache, q, at, "f32", workspace=(one, need))
            b = run_attention(dev, cache, q, at, "f32")
            assert np.isfinite(a).all() and np.array_equal(a.view(np.uint32), b.view(np.uint32)), (T, H, at)
        assert not dev.get(one, WORKSPACE_ZERO, np.uint8).any()


def test_two_streams_with_workspaces_of_their_own(hip_ctx):
    import ctypes as C
    rng = np.random.default_rng(18)
    n, T, H = 5000, 1, 12
    k, v = rows(rng, n, 3, 64, "f32"), rows(rng, n, 3, 64, "f32")
    cache = Q4Cache(hip_ctx, 3, n, 64)
    streams = [C.c_void_p() for _ in range(2)]
    for s in streams:
        L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(s)))
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        need = cache.workspace_bytes(T, H, n - 1)
        assert need
        qs = [rows(rng, T, H, 64, "f32") for _ in streams]
        want = [run_attention(dev, cache, q, n - 1, "f32") for q in qs]
        ws, outs, qp = [(dev.empty(need, 0), need) for _ in streams], [dev.empty(T * H * 64 * 4) for _ in streams], \
            [dev.put(q) for q in qs]
        for _ in range(50):
            for s, w, o, q in zip(streams, ws, outs, qp):
                cache.attention(q, o, T, H, n - 1, workspace=w, stream=s)
        for s in streams:
            L.check(L.lib().ahip_stream_synchronize(s))
        for o, w in zip(outs, want):
            assert np.array_equal(dev.get(o, w.shape, np.float32).view(np.uint32), w.view(np.uint32))
    for s in streams:
        L.check(L.lib().ahip_stream_destroy(s))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_at_any_element_and_stride(hip_ctx, dtype):
    """Rows one element past a wide load's alignment, strides odd: the same bits as of aligned rows."""
    rng = np.random.default_rng(19)
    T, H, KVH, hd, size = 37, 6, 2, 64, NP[dtype]().nbytes
    w, wk = H * hd, KVH * hd
    q, k, v = rows(rng, T, H, hd, dtype), rows(rng, T, KVH, hd, dtype), rows(rng, T, KVH, hd, dtype)
    table, gain = rope_table(T, hd, 1e4), (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)

    def shifted(dev, x):
        flat, stride = padded(x, 1)
        return dev.put(np.concatenate([np.zeros(1, x.dtype), flat.reshape(-1)])) + size, stride

    def taken(dev, p, width):
        return dev.get(p, (T, width + 1), NP[dtype])[:, :width]

    with ref.Device(hip_ctx) as dev:
        got = []
        for odd in (False, True):
            cache = Q4Cache(hip_ctx, KVH, T, hd)
            put = shifted if odd else (lambda dev, x: (dev.put(x), x[0].size))
            (qp, qs), (kp, ks), (vp, vs) = put(dev, q), put(dev, k), put(dev, v)
            g, tab = dev.put(gain), dev.put(table)
            o = [dev.empty((T + 1) * (n + 1) * size) + (size if odd else 0) for n in (w, wk, wk, wk, w)]
            n = 1 if odd else 0
            qk_norm_rope(hip_ctx, qp, kp, T, H, KVH, hd, o[0], o[1], dtype, g, g, 1e-6, tab, T, q_stride=qs,
                         k_stride=ks, q_out_stride=w + n, k_out_stride=wk + n)
            cache.store(kp, vp, T, 0, dtype, ks, vs)
            cache.load(o[2], o[3], T, 0, dtype, wk + n, wk + n)
            cache.attention(qp, o[4], T, H, 0, dtype, qs, w + n)
            got.append([taken(dev, p, n) if odd else dev.get(p, (T, n), NP[dtype])
                        for p, n in zip(o, (w, wk, wk, wk, w))])
    for a, b in zip(*got):
        assert np.isfinite(a.astype(np.float64)).all() and np.array_equal(a, b)


def test_offsets_past_32_bits(hip_ctx):
    """A head's cache of 4.8 GB, and rows 4 GiB elements apart.

    All keys but 40 are zeros, of score 0; the query scores 60 or more with one of the 40, so that the others' share
    is below 2^25 e^-60 < 2^-61 and the 40 alone, closed up, are the reference."""
    rng = np.random.default_rng(20)
    cap, hd, n = 1 << 25, 256, 40
    at = np.array([5, (1 << 24) - 7, cap - 20])  # 12, 12 and 16 rows from there
    sizes = (12, 12, 16)
    k, v = rows(rng, n, 2, hd, "f16"), rows(rng, n, 2, hd, "f16")
    q = (k[-1:] * 8).astype(np.float32)  # the last key's own: a score near 8 * 256 / 16 = 128
    far = 1 << 31
    cache = Q4Cache(hip_ctx, 2, cap, hd)
    assert cache.bytes // 4 > 1 << 32
    with ref.Device(hip_ctx) as dev:
        for p in (cache._desc.k, cache._desc.v):
            L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0, cache.bytes // 2))
        a = 0
        for start, m in zip(at, sizes):
            store(dev, cache, k[a:a + m], v[a:a + m], int(start), "f16")
            a += m
        kd, vd = ref.q4_rows(k.astype(np.float32), v.astype(np.float32))
        a = 0
        for start, m in zip(at, sizes):
            got = load(dev, cache, int(start) - 2 if a else 0, m + 2 if a else m, "f32")
            if a:
                assert all((g[:2] == 0).all() for g in got)
                assert equal(got[0][2:], kd[a:a + m]) and equal(got[1][2:], vd[a:a + m])
            a += m
        # the last 4 positions are behind the query's
        got = run_attention(dev, cache, q, cap - 5, "f32")
        q2 = (k[-5:-4] * 8).astype(np.float32)
        own = run_attention(dev, cache, q2, cap - 5, "f32")
        # three rows of two heads, 2^31 elements (4 GiB of f16) from one to the next
        w = 2 * hd
        src, dst = dev.empty(2 * (2 * far + w)), dev.empty(2 * (2 * far + w))
        for i in range(3):
            L.check(L.lib().ahip_memcpy_htod(hip_ctx.handle, src + 2 * far * i, k[i:i + 1].ctypes.data, 2 * w))
        cache.store(src, src, 3, 100, "f16", far, far)
        cache.load(dst, None, 3, 100, "f16", far, far)
        for i in range(3):
            assert np.array_equal(dev.get(dst + 2 * far * i, (2, hd), np.float16), kd[i].astype(np.float16)), i
        qk_norm_rope(hip_ctx, src, None, 3, 2, 0, hd, dst, None, "f16", q_stride=far, q_out_stride=far)
        for i in range(3):
            assert np.array_equal(dev.get(dst + 2 * far * i, (2, hd), np.float16), k[i]), i
        cache.attention(src, dst, 3, 2, 0, "f16", far, far)  # positions 0 to 2: zeros
        for i in range(3):
            assert not dev.get(dst + 2 * far * i, (2, hd), np.float16).any(), i
    cache.close()
    score = (kd[:n - 4, :] * q2[0]).sum(-1).max(0) / 16
    assert (score > 60).all()
    check_attention(own, q2, kd[:n - 4], vd[:n - 4], n - 5, "f32", "far")
    assert np.isfinite(got).all()


# ---------------------------------------------------------------- norm and rotation

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", [
    (9, 3, 64, 1, 2000), (32, 8, 128, 33, 0), (1, 0, 32, 5, 3), (0, 2, 96, 7, 1), (3, 1, 160, 2, 9), (2, 2, 192, 3, 0),
    (5, 1, 224, 1, 0), (4, 4, 256, 65, 100)])
def test_norm_and_rotation(hip_ctx, heads, kv_heads, hd, tokens, start, interleaved, dtype):
    rng = np.random.default_rng(hd + tokens)
    t = NP[dtype]
    table = rope_table(start + tokens, hd, 1e5)
    with ref.Device(hip_ctx) as dev:
        dtab = dev.put(table)
        for norm, rope, extra in ((True, True, 0), (True, False, 8), (False, True, 3), (False, False, 1)):
            x = {"q": rows(rng, tokens, heads, hd, dtype, 2), "k": rows(rng, tokens, kv_heads, hd, dtype, 0.01)}
            gain = {n: (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if norm else None for n in x}
            arg = {}
            for n in x:
                p, s = padded(x[n], extra)
                arg[n], arg[n + "_stride"] = dev.put(p), s
                arg[n + "_out"] = dev.empty(max(1, tokens * s * p.itemsize))
                arg[n + "_out_stride"] = s
                arg[n + "_gain"] = dev.put(gain[n]) if norm else None
            qk_norm_rope(hip_ctx, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=hd, dtype=dtype, eps=1e-5,
                         rope=dtab if rope else None, rope_positions=len(table), interleaved=interleaved, start=start,
                         **arg)
            for n, y in x.items():
                if not y.size:
                    continue
                got = dev.get(arg[n + "_out"], (tokens, arg[n + "_stride"]), t)
                if extra:
                    assert (got[:, -extra:].view(np.uint8) == 0xA5).all()
                got = got[:, :y[0].size].reshape(y.shape).astype(np.float64)
                want = ref.norm_rope(y, gain[n], 1e-5, table[start:] if rope else None, interleaved)
                # the norm loses half a float32 step for each of its hd squares and their sums (half of that in the
                # root) and a few more; the rotation three of the pair's larger value
                pair = np.abs(ref.norm_rope(y, gain[n], 1e-5, None, interleaved))
                pair = np.maximum(pair, np.roll(pair, hd // 2, -1) if not interleaved else
                                  pair.reshape(*y.shape[:2], -1, 2)[..., ::-1].reshape(y.shape))
                bound = ((hd / 2 + 6) * norm + 6 * rope) * ref.EPS32 * pair
                if dtype == "f16":
                    bound = bound * (1 + ref.EPS16) + ref.EPS16 * np.abs(want) + 2.0 ** -25
                assert (np.abs(got - want) <= bound).all(), (n, norm, rope)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_norm_and_rotation_in_place_and_at_given_positions(hip_ctx, dtype):
    rng = np.random.default_rng(21)
    t = NP[dtype]
    table = rope_table(50, 64, 1e4)
    pos = np.array([49, 0, 7, 7, 50, -1, 12], np.int32)
    stacked = rows(rng, 7, 6, 64, dtype)  # [q 3 | k 1 | v 2]
    gain = np.ones(64, np.float32)
    with ref.Device(hip_ctx) as dev:
        p, g = dev.put(stacked), dev.put(gain)
        qk_norm_rope(hip_ctx, p, p + 3 * 64 * stacked.itemsize, 7, 3, 1, 64, p, p + 3 * 64 * stacked.itemsize, dtype,
                     g, g, 1e-6, dev.put(table), 50, positions=dev.put(pos), q_stride=384, k_stride=384,
                     q_out_stride=384, k_out_stride=384)
        got = dev.get(p, (7, 6, 64), t)
    assert np.array_equal(got[:, 4:], stacked[:, 4:])
    outside = (pos < 0) | (pos >= 50)
    assert np.isnan(got[outside, :4]).all()
    want = ref.norm_rope(stacked[:, :4], gain, 1e-6, table[np.where(outside, 0, pos)], True)
    off = np.abs(got[:, :4] - want)[~outside]
    assert off.max() <= (ref.EPS16 if dtype == "f16" else 48 * ref.EPS32) * 8 * 1.001  # no value past sqrt(64) = 8


def test_norm_of_zeros_and_of_non_finite_values(hip_ctx):
    x = np.zeros((4, 2, 64), np.float32)
    x[1, 0, 3], x[2, 1, 5] = np.nan, np.inf
    with ref.Device(hip_ctx) as dev:
        p, o = dev.put(x), dev.empty(x.nbytes)
        qk_norm_rope(hip_ctx, p, None, 4, 2, 0, 64, o, None, q_gain=dev.put(np.ones(64, np.float32)))
        got = dev.get(o, x.shape, np.float32)
    assert np.isnan(got[1, 0]).all() and np.isnan(got[2, 1, 5])
    keep = np.ones((4, 2), bool)
    keep[1, 0] = keep[2, 1] = False
    assert (got[keep] == 0).all() and (np.delete(got[2, 1], 5) == 0).all()


# ---------------------------------------------------------------- together, on a stream

def test_a_layer_s_steps_together_on_a_stream(hip_ctx):
    """Norm and rotation, store and attention of a prompt, then of single tokens, queued on a stream without waits."""
    import ctypes as C
    rng = np.random.default_rng(31)
    H, KVH, hd, lens = 6, 2, 64, [50, 1, 1, 7, 1]
    cap = sum(lens)
    table, gain = rope_table(cap, hd, 1e5), (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    qkv = rows(rng, cap, H + 2 * KVH, hd, "f32", 2)
    stream = C.c_void_p()
    L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(stream)))
    cache = Q4Cache(hip_ctx, KVH, cap, hd)
    w = (H + 2 * KVH) * hd
    with ref.Device(hip_ctx) as dev:
        p, g, tab, out = dev.put(qkv), dev.put(gain), dev.put(table), dev.empty(cap * H * hd * 4)
        work = max(cache.workspace_bytes(n, H, sum(lens[:i])) for i, n in enumerate(lens))
        ws = (dev.empty(max(work, 1), 0), work)
        at = 0
        for n in lens:
            row = p + at * w * 4
            k, v = row + H * hd * 4, row + (H + KVH) * hd * 4
            qk_norm_rope(hip_ctx, row, k, n, H, KVH, hd, row, k, q_gain=g, k_gain=g, rope=tab, rope_positions=cap,
                         start=at, q_stride=w, k_stride=w, q_out_stride=w, k_out_stride=w, stream=stream)
            cache.store(k, v, n, at, k_stride=w, v_stride=w, stream=stream)
            cache.attention(row, out + at * H * hd * 4, n, H, at, q_stride=w, workspace=ws, stream=stream)
            at += n
        L.check(L.lib().ahip_stream_synchronize(stream))
        got, rotated = dev.get(out, (cap, H, hd), np.float32), dev.get(p, (cap, H + 2 * KVH, hd), np.float32)
    L.check(L.lib().ahip_stream_destroy(stream))
    want = ref.norm_rope(qkv[:, :H + KVH], gain, 1e-5, table, True)
    assert np.abs(rotated[:, :H + KVH] - want).max() <= 48 * ref.EPS32 * 3 * 8
    # the attention from the rows that the kernel rotated: the quantiser may round a value on a border either way
    check_attention(got, rotated[:, :H], *ref.q4_rows(rotated[:, H:H + KVH], rotated[:, H + KVH:]), 0, "f32", "layer")
