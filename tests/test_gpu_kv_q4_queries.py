"""Queries at the ends of their types over the 4-bit KV cache, in every kernel
of the attention: scores past the integers that float32 holds, and queries that
are no numbers."""
import numpy as np
import pytest

from alpaca_amd.kvcache import Q4Cache
from tests import q4_reference as ref
from tests.test_gpu_kv_q4 import NP, run_attention, rows, store

pytestmark = pytest.mark.gpu

# (heads, kv_heads, head_dim, tokens, positions before them)
SHAPES = [(16, 1, 32, 1, 70), (8, 2, 64, 1, 299), (4, 1, 128, 1, 3000), (2, 1, 256, 1, 90),  # single tokens
          (6, 2, 64, 5, 200), (17, 1, 128, 3, 1500), (4, 2, 256, 40, 33),  # 16 columns a workgroup
          (400, 200, 32, 90, 5),  # 32, of float32; of f16 many
          (128, 128, 128, 250, 37), (64, 64, 160, 250, 3), (130, 130, 64, 70, 1600), (200, 200, 128, 250, 200)]


@pytest.mark.parametrize("dtype,size", [("f32", 1e4), ("f32", 6e4), ("f32", 1e15), ("f16", 1e4), ("f16", 6e4)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", SHAPES)
def test_large_scores(hip_ctx, heads, kv_heads, hd, tokens, start, sign, dtype, size):
    """Keys along the queries, from one to two times 30,000 in the order of their positions: scores of 1e9 and more,
    whose neighbours are the same bits or half an f16 step, 2^-12, apart: the last key's, or for queries of the other
    sign the first one's, takes all of the weight, with those of its bits."""
    rng = np.random.default_rng(heads + hd + start)
    n = start + tokens
    u = rng.choice([-1.0, 1.0], hd)
    b = 30000 * (1 + np.arange(n) / n)
    k = np.broadcast_to(b[:, None, None] * u, (n, kv_heads, hd)).astype(np.float32)
    v = rows(rng, n, kv_heads, hd, "f32")
    q = np.broadcast_to(sign * size * u, (tokens, heads, hd)).astype(NP[dtype])
    cache = Q4Cache(hip_ctx, kv_heads, n + 5, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, start, dtype).astype(np.float64)
    cache.close()
    kd, vd = ref.q4_rows(k, v)
    score = kd[:, 0] @ (sign * u)  # the same for all heads
    assert np.isfinite(got).all()
    for t in {*range(0, tokens, max(1, tokens // 9)), tokens - 1}:
        seen = score[:start + t + 1]
        top = seen == seen.max()
        assert (seen[~top] < seen.max() - 2.0 ** -12 * np.abs(seen).max()).all()
        want = np.repeat(vd[:len(seen)][top].mean(0), heads // kv_heads, 0)
        # weights of 1 and 0: the sums' roundings and, in f16, half a step of the values and of the output
        most = np.abs(vd).max()
        bound = (top.sum() + 64) * ref.EPS32 * most + (2 * ref.EPS16 * most + 2.0 ** -24) * (dtype == "f16")
        assert (np.abs(got[t] - want) <= bound).all(), t


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", SHAPES)
def test_a_query_that_is_no_number_reaches_its_own_output_only(hip_ctx, heads, kv_heads, hd, tokens, start, value,
                                                               dtype):
    rng = np.random.default_rng(heads + hd + start + 1)
    n = start + tokens
    k, v = rows(rng, n, kv_heads, hd, "f32"), rows(rng, n, kv_heads, hd, "f32")
    q = rows(rng, tokens, heads, hd, dtype)
    hit = (tokens // 2, heads // 2)
    bad = q.copy()
    bad[hit][hd - 3] = value
    cache = Q4Cache(hip_ctx, kv_heads, n, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        want, got = (run_attention(dev, cache, x, start, dtype) for x in (q, bad))
    cache.close()
    assert np.isfinite(want).all() and np.isnan(got[hit]).all()
    got[hit] = want[hit]
    assert np.array_equal(got, want)
