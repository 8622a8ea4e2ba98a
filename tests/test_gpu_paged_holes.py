"""Attention over pages where the table has a hole: a page that there is not gives NaN to the queries that see one of
its positions and changes nothing for the others, whatever lies in the pages that no table names."""
import numpy as np
import pytest

from tests import paged_reference as ref
from tests.paged_reference import Batch
from tests.q4_reference import Device
from tests.test_gpu_paged import attend, fill, make, rows

pytestmark = pytest.mark.gpu

# (heads, kv_heads, hd, new tokens, position of the first, tokens of a workgroup's columns): workgroups of few
# columns, of 64, 128 and 256, and of 64 whose steps are shared
SHAPES = [(4, 4, 64, 60, 24, 16), (64, 64, 64, 250, 8, 64), (32, 32, 128, 250, 8, 64), (32, 8, 128, 200, 3032, 16),
          (64, 64, 32, 300, 40, 128), (64, 64, 64, 300, 40, 128), (64, 64, 96, 300, 40, 128), (64, 64, 160, 300, 40, 128),
          (64, 64, 256, 300, 40, 128), (64, 64, 64, 700, 8, 128), (64, 64, 96, 1700, 8, 256), (64, 64, 128, 1700, 8, 256)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_hole_reaches_only_the_queries_that_see_it(hip_ctx, shape, window, sinks, dtype):
    """The hole begins inside a step of 32 keys, behind the last position of a workgroup's queries; page 0 is no one's and
    holds NaN."""
    heads, kv_heads, hd, new, first, each = shape
    rng = np.random.default_rng(heads + hd + new)
    n = first + new
    b = Batch(rng, 16, [new], [n], pages=-(-n // 16) + 3)
    spare = min(set(range(1, b.pages)) - set(b.table.ravel().tolist()))
    b.table[b.table == 0] = spare
    last = first + each - 1
    hole = last // 16 + 1
    assert last % 32 < 16 and hole * 16 < n
    q = rows(rng, new, heads, hd, dtype)
    cache = make(hip_ctx, b, kv_heads, hd)
    some = [0, heads - 1]
    pos = np.arange(first, n)
    sees_it = (pos >= hole * 16) & ((pos < hole * 16 + 15 + window) if window else True)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        for entry in (-1, b.pages):
            b.table[0, hole] = entry
            got = attend(dev, cache, b.on(dev), q, dtype, window=window, sinks=sinks)
            assert np.array_equal(np.isnan(got).any((1, 2)), sees_it), (entry, np.flatnonzero(np.isnan(got).any((1, 2)) != sees_it))
            assert np.isnan(got[sees_it]).all()
            want, bound = ref.attention(q, *data[0], first, dtype, window, sinks, heads=some)
            near = np.abs(got.astype(np.float64) - want) <= bound
            assert near[:, some][~sees_it].all()
    cache.close()
