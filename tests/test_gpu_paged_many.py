"""Batches of thousands of sequences over pages, most of few tokens and some without rows."""
import numpy as np
import pytest

from alpaca_amd.kvcache import rope_table
from tests import paged_reference as ref
from tests.paged_reference import Batch
from tests.q4_reference import Device
from tests.test_gpu_paged import Rows, append, attend, load, make, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,chunk,window", [(4, 0, 0), (4, 0, 20), (64, 300, 0)])
def test_thousands_of_sequences(hip_ctx, heads, chunk, window, dtype):
    rng = np.random.default_rng(heads + window)
    S, KVH, hd, page = 3001, heads // 2, 64, 16
    lengths = [int(n) for n in rng.integers(1, 50, S)]
    new = [int(min(n, rng.integers(0, 3))) for n in lengths]
    if chunk:
        lengths[2000], new[2000] = chunk + 100, chunk
    b = Batch(rng, page, new, lengths)
    table = rope_table(max(lengths), hd, 1e4)
    cache = make(hip_ctx, b, KVH, hd)
    some = [0, heads - 1]
    with Device(hip_ctx) as dev:
        w = ref.whole(rng, b)
        k, v = (rows(rng, w.rows, KVH, hd, "f16") for _ in range(2))
        append(dev, cache, w.on(dev), k, v, "f16")
        q, nk, nv = (rows(rng, b.rows, n, hd, dtype) for n in (heads, KVH, KVH))
        out, on = Rows(dev, b.rows, heads * hd, dtype), b.on(dev)
        append(dev, cache, on, nk, nv, dtype, q=dev.put(q), q_out=out.p, heads=heads, rope=dev.put(table),
               rope_positions=len(table))
        turned, (got_k, got_v) = out.get(heads), load(dev, cache, on, b.rows, "f16")
        got = attend(dev, cache, on, turned, dtype, window=window, sinks=window and 2)
    cache.close()
    pos = np.array([p for _, p in b.positions()])
    for x, y, t in ((q, turned, dtype), (nk, got_k, "f16")):
        want, off = ref.rotated(x, pos, table, True)
        assert (np.abs(y - want) <= off + ref.half_step(np.abs(want) + off, t)).all()
    assert np.array_equal(got_v, nv.astype(np.float16))
    for s in range(S):
        r, n = b.sequence_rows(s), b.lengths[s] - b.new[s]
        held = [np.concatenate([x[w.sequence_rows(s)][:n], y[r]]) for x, y in ((k, got_k), (v, got_v))]
        want, bound = ref.attention(turned[r], *held, n, dtype, window, window and 2, heads=some)
        assert (np.abs(got[r].astype(np.float64) - want) <= bound)[:, some].all(), s
