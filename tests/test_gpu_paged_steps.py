"""Whole steps over a KV cache in pages: append, attention and log probabilities
of a batch as a serving loop runs them, eagerly and as a captured graph whose
batch changes between replays; and pages past 32-bit offsets."""
import ctypes as C

import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd.kvcache import PAGED_WORKSPACE_ZERO, PagedBatch, PagedCache, rope_table
from alpaca_amd.sampling import LOGPROBS_WORKSPACE_ZERO, token_logprobs
from tests import paged_reference as ref
from tests.paged_reference import NP, Batch
from tests.q4_reference import Device
from tests.test_gpu_kv_q4_graph import capture
from tests.test_gpu_paged import append, attend, garbage, load, make, rows

pytestmark = pytest.mark.gpu


def put(ctx, p, a):
    a = np.ascontiguousarray(a)
    L.check(L.lib().ahip_memcpy_htod(ctx.handle, p, a.ctypes.data, a.nbytes))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,page,window,sinks", [(9, 3, 64, 16, 0, 0), (8, 2, 128, 32, 40, 3)])
def test_a_serving_loop(hip_ctx, heads, kv_heads, hd, page, window, sinks, dtype):
    """Conversations that start with prompts, decode, end and give their pages to new ones: every step's attention against
    all that was said so far."""
    rng = np.random.default_rng(hd)
    pages, stride, most = 40, 20, 300
    table = rope_table(most, hd, 1e4)
    cache = PagedCache(hip_ctx, pages, kv_heads, hd, page)
    garbage(hip_ctx, cache)
    free, said, held = list(rng.permutation(pages)), {}, {}  # rows and pages by conversation
    new_ones = iter(range(1000))
    with Device(hip_ctx) as dev:
        tab = dev.put(table)
        for step in range(30):
            if len(said) < 5 and len(free) > 8 and step % 2 == 0:
                c = next(new_ones)
                said[c], held[c] = (np.zeros((0, kv_heads, hd), np.float16),) * 2, []
            for c in [c for c in said if len(said[c][0]) > 60 and step % 7 == 3]:
                free += held.pop(c)
                del said[c]
            order = list(rng.permutation(list(said)))
            new = [int(rng.integers(1, 30)) if len(said[c][0]) == 0 else int(rng.integers(0, 3)) for c in order]
            lengths = [len(said[c][0]) + m for c, m in zip(order, new)]
            b = Batch(rng, page, new, lengths, pages, spare_rows=step % 3, stride=stride)
            for s, c in enumerate(order):
                while len(held[c]) * page < lengths[s]:
                    held[c].append(free.pop())
                b.table[s] = -1
                b.table[s, :len(held[c])] = held[c]
            q, k, v = (rows(rng, b.rows, n, hd, dtype) for n in (heads, kv_heads, kv_heads))
            on, place = b.on(dev, step % 2 == 0), dev.put(q)
            append(dev, cache, on, k, v, dtype, q=place, q_out=place, heads=heads, rope=tab, rope_positions=most)
            turned = dev.get(place, q.shape, q.dtype)
            mine = slice(0, b.starts[-1])
            pos = np.array([p for _, p in b.positions()], int)
            want, off = ref.rotated(q[mine], pos, table, True)
            assert (np.abs(turned[mine].astype(np.float64) - want) <= off + ref.half_step(np.abs(want) + off, dtype)).all()
            got_k, got_v = load(dev, cache, on, b.rows, "f16")
            out = attend(dev, cache, on, turned, dtype, window=window, sinks=sinks)
            for s, c in enumerate(order):
                r = b.sequence_rows(s)
                assert np.array_equal(got_v[r], v[r].astype(np.float16))
                # the keys as they were read back (their rotation is checked with the queries')
                said[c] = tuple(np.concatenate(x) for x in zip(said[c], (got_k[r], got_v[r])))
                want, off = ref.rotated(k[r], pos[r], table, True)
                assert (np.abs(got_k[r] - want) <= off + ref.half_step(np.abs(want) + off, "f16")).all()
                want, bound = ref.attention(turned[r], *said[c], lengths[s] - new[s], dtype, window, sinks)
                assert (np.abs(out[r].astype(np.float64) - want) <= bound).all(), (step, s)
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,window", [(9, 3, 64, 0), (8, 2, 128, 200), (64, 64, 64, 0)])
def test_a_captured_step_follows_its_batch(hip_ctx, heads, kv_heads, hd, window, dtype):
    """Append, attention and log probabilities of a fixed number of rows in a graph; row starts, lengths and pages change
    between replays, with the program's eager calls between."""
    rng = np.random.default_rng(heads)
    page, stride, pages, S, T, vocab = 32, 90, 400, 4, 330, 5000
    t = NP[dtype]
    w, wk, size = heads * hd, kv_heads * hd, t().nbytes
    table = rope_table(stride * page, hd, 1e5)
    stream = C.c_void_p()
    L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(stream)))
    caches = [PagedCache(hip_ctx, pages, kv_heads, hd, page) for _ in range(2)]
    old = [rows(rng, pages * page, kv_heads, hd, "f16") for _ in range(2)]
    with Device(hip_ctx) as dev:
        n = pages * page
        every = PagedBatch(dev.put(np.array([0, n], np.int32)), dev.put(np.array([n], np.int32)),
                           dev.put(np.arange(pages, dtype=np.int32)), 1, pages, n, n)
        for c in caches:
            append(dev, c, every, *old, "f16")
        arrays = [dev.empty(4 * x) for x in (S + 1, S, S * stride)]
        on = PagedBatch(*arrays, S, stride, T, 0)
        tab = dev.put(table)
        q, k, v, qr, out = (dev.empty(T * x * size) for x in (w, wk, wk, w, w))
        need = caches[0].workspace_bytes()
        works = [(dev.empty(need, 0), need) for _ in range(2)]
        lneed = C.c_int64()
        L.check(L.lib().ahip_token_logprobs_workspace(C.byref(lneed)))
        lworks = [(dev.empty(lneed.value, 0), lneed.value) for _ in range(2)]
        logits, tokens = dev.empty(3 * vocab * 4), dev.empty(12)
        answers = [dev.empty(x) for x in (12, 12, 3 * 7 * 4, 3 * 7 * 4)]

        def step(cache, work, lwork, s):
            cache.append(on, k, v, q, qr, heads, dtype, rope=tab, rope_positions=len(table), stream=s)
            cache.attention(on, qr, out, heads, dtype, window=window, sinks=window and 5, workspace=work, stream=s)
            token_logprobs(hip_ctx, logits, 3, vocab, tokens, answers[0], answers[1], 7, answers[2], answers[3],
                           workspace=lwork, stream=s)
        launch, destroy = capture(stream, lambda: step(caches[0], works[0], lworks[0], stream))

        def results():
            got = [dev.get(p, (T, heads, hd), t) for p in (qr, out)]
            got += [dev.get(p, (3, m), d) for p, m, d in zip(answers, (1, 1, 7, 7), (np.float32,) * 2 + (np.int32, np.float32))]
            for p in (qr, out):
                L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0xA5, T * w * size))
            for p in answers:
                L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0xA5, 12))
            return got
        for i, (new, lengths) in enumerate([([1, 1, 1, 1], [5, 2800, 40, 64]), ([300, 20, 0, 10], [300, 1000, 7, 2000]),
                                            ([0, 0, 0, 0], [0, 0, 0, 0]), ([1, 325, 1, 3], [2000, 2000, 1, 3]),
                                            ([2, 2, 2, 2], [2500, 2500, 2500, 2500]), ([1, 1, 1, 1], [6, 2801, 41, 65])]):
            b = Batch(rng, page, new, lengths, pages, stride=stride)
            for p, a in zip(arrays, (b.starts, b.lengths, b.table)):
                put(hip_ctx, p, np.array(a, np.int32))
            for p, m in ((q, heads), (k, kv_heads), (v, kv_heads)):
                put(hip_ctx, p, rows(rng, T, m, hd, dtype))
            put(hip_ctx, logits, rng.standard_normal((3, vocab)).astype(np.float32))
            put(hip_ctx, tokens, rng.integers(0, vocab, 3).astype(np.int32))
            results()
            launch()
            got = results()
            step(caches[1], works[1], lworks[1], None)  # the program's own eager work, on its own cache
            want = results()
            used = b.starts[-1]
            assert np.isfinite(want[1][:used].astype(np.float32)).all() and (want[1][used:].view(np.uint8) == 0xA5).all()
            assert all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(got, want)), i
            # and a call of another shape over the graph's cache, with the cache's own workspace
            other = Batch(rng, page, [3, 1], [900, 2000], pages, stride=stride)
            attend(dev, caches[0], other.on(dev), rows(rng, 4, heads, hd, dtype), dtype)
        data = [dev.get(p, c.bytes // 2, np.uint8) for c in caches for p in (c._desc.k, c._desc.v)]
        assert np.array_equal(data[0], data[2]) and np.array_equal(data[1], data[3])
        assert not any(dev.get(p, PAGED_WORKSPACE_ZERO, np.uint8).any() for p, _ in works)
        assert not any(dev.get(p, LOGPROBS_WORKSPACE_ZERO, np.uint8).any() for p, _ in lworks)
        destroy()
    L.check(L.lib().ahip_stream_destroy(stream))
    for c in caches:
        c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_pages_past_32_bit_offsets(hip_ctx, dtype):
    """Pages of a cache of more than 4 GiB, spread over all of it: sequences of few columns and of many."""
    rng = np.random.default_rng(23)
    KVH, hd, page, pages = 4, 128, 1024, 4200
    cache = PagedCache(hip_ctx, pages, KVH, hd, page)
    assert cache.bytes // 2 > 1 << 32
    b = Batch(rng, page, [1, 300], [2500, 2100], pages)
    b.table[0], b.table[1] = [0, pages - 1, 2048], [pages - 2, 2049, 4100]
    garbage(hip_ctx, cache)
    with Device(hip_ctx) as dev:
        w = ref.whole(rng, b)
        k, v = (rows(rng, w.rows, KVH, hd, "f16") for _ in range(2))
        append(dev, cache, w.on(dev), k, v, "f16")
        assert all(np.array_equal(x, y) for x, y in zip(load(dev, cache, w.on(dev), w.rows, "f16"), (k, v)))
        for heads in (4, 64):
            q = rows(rng, b.rows, heads, hd, dtype)
            got = attend(dev, cache, b.on(dev), q, dtype)
            for s in range(2):
                r, some = b.sequence_rows(s), [0, heads - 1]
                want, bound = ref.attention(q[r], k[w.sequence_rows(s)], v[w.sequence_rows(s)], b.lengths[s] - b.new[s],
                                            dtype, heads=some)
                assert (np.abs(got[r].astype(np.float64) - want) <= bound)[:, some].all()
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_page_is_copied_by_its_bytes(hip_ctx, dtype):
    """A conversation that forks: its last page's bytes copied to a page of its own."""
    rng = np.random.default_rng(24)
    b = Batch(rng, 32, [1, 1], [71, 71])
    cache = make(hip_ctx, b, 2, 64)
    b.table[1, :2] = b.table[0, :2]
    with Device(hip_ctx) as dev:
        k, v = (rows(rng, 70, 2, 64, "f16") for _ in range(2))
        first = Batch(rng, 32, [70], [70], b.pages, stride=b.stride)
        first.table = b.table[:1]
        append(dev, cache, first.on(dev), k, v, "f16")
        n, src, dst = cache.bytes // 2 // b.pages, int(b.table[0, 2]), int(b.table[1, 2])
        stream = C.c_void_p()
        L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(stream)))
        for p in (cache._desc.k, cache._desc.v):
            L.check(L.lib().ahip_memcpy_dtod_async(p + dst * n, p + src * n, n, stream))
        L.check(L.lib().ahip_stream_synchronize(stream))
        L.check(L.lib().ahip_stream_destroy(stream))
        more = [rows(rng, 2, 2, 64, "f16") for _ in range(2)]
        append(dev, cache, b.on(dev), *more, "f16")
        q = rows(rng, 2, 4, 64, dtype)
        got = attend(dev, cache, b.on(dev), q, dtype)
        for s in range(2):
            ks, vs = (np.concatenate([x, y[s:s + 1]]) for x, y in zip((k, v), more))
            want, bound = ref.attention(q[s:s + 1], ks, vs, 70, dtype)
            assert (np.abs(got[s:s + 1].astype(np.float64) - want) <= bound).all()
    cache.close()
