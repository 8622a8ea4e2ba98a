"""Attention over a 4-bit cache whose offsets pass 32 bits: rows far apart that
share a query's weight, and rows behind it that would take all of it."""
import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd.kvcache import Q4Cache
from tests import q4_reference as ref
from tests.test_gpu_kv_q4 import NP, check_attention, run_attention, store

pytestmark = pytest.mark.gpu


def test_rows_far_apart_share_the_weight(hip_ctx):
    """All keys but 40 are zeros, of score 0.  36 rows, 12 each near the start, past 4 GiB and near the end, have scores
    of some 80 +- 2 and the 4 behind the queries of 100 and more: the zeros' share is below 2^25 e^-70 < 2^-75, and the
    rows alone, closed up, are the reference."""
    rng = np.random.default_rng(22)
    cap, hd, KVH = 1 << 25, 256, 2
    places, sizes = (5, (1 << 24) - 7, cap - 20), (12, 12, 16)
    n = sum(sizes)
    u = rng.choice([-1.0, 1.0], (KVH, hd))
    size = np.where(np.arange(n) < 36, 1 + 0.02 * rng.standard_normal(n), 1.3)[:, None, None]
    k = (size * u + 0.05 * rng.standard_normal((n, KVH, hd))).astype(np.float32)
    v = rng.standard_normal((n, KVH, hd)).astype(np.float32)
    kd, vd = ref.q4_rows(k, v)
    cache = Q4Cache(hip_ctx, KVH, cap, hd)
    assert cache.bytes // 2 // KVH > 1 << 32
    with ref.Device(hip_ctx) as dev:
        for p in (cache._desc.k, cache._desc.v):
            L.check(L.lib().ahip_memset(hip_ctx.handle, p, 0, cache.bytes // 2))
        a = 0
        for start, m in zip(places, sizes):
            store(dev, cache, k[a:a + m], v[a:a + m], start, "f32")
            a += m
        # one query of a head (a single token's kernel), four of two heads, and rows of nine
        for T, H, dtype in ((1, 2, "f32"), (1, 2, "f16"), (2, 4, "f32"), (9, 2, "f32"), (9, 2, "f16"), (9, 6, "f32")):
            q = (5 * np.repeat(u, H // KVH, 0) * (1 + 0.01 * rng.standard_normal((T, H, 1)))).astype(NP[dtype])
            first = 36 - T  # in the rows closed up; the last query is at cap - 9
            score = np.einsum("thd,nhd->tnh", q.astype(np.float64), np.repeat(kd, H // KVH, 1)) / 16
            assert (score[:, :36] > 70).all() and (score[:, 36:] > score[:, :36].max() + 5).all()
            p = np.exp(score[:, :36] - score[:, :36].max())
            assert all((p[:, i:i + 12].sum(1) > 0.02 * p.sum(1)).all() for i in (0, 12, 24))  # no place holds all of it
            for dev_start in (False, True):
                kw = {"start_dev": dev.put(np.array([cap - 8 - T], np.int32))} if dev_start else {}
                got = run_attention(dev, cache, q, 0 if dev_start else cap - 8 - T, dtype, **kw)
                check_attention(got, q, kd[:36], vd[:36], first, dtype, (T, H, dtype, dev_start))
    cache.close()
