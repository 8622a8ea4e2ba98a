"""Scores so large that neighbouring float32 numbers are several apart: the probabilities of a step whose largest score
is one such number past the earlier ones stay inside f16."""
import numpy as np
import pytest

from tests import paged_reference as ref
from tests.paged_reference import NP, Batch
from tests.q4_reference import Device
from tests.test_gpu_paged import append, attend, make

pytestmark = pytest.mark.gpu


def large_scores(band, count):
    """(x0, x1): scores, exact in float32, whose base-2 forms x log2(e) / 8 lie in [2^band, 2^(band + 1)) and are 8 apart
    once rounded, with m + 6 rounded no less than the larger."""
    f = np.float32
    sc = f(1.4426950408889634) / f(8)
    found = []
    for j in range(int(2.0 ** band / sc / 32) + 2, int(2.0 ** (band + 1) / sc / 32) - 2, 997):
        x0, x1 = 32 * j, 32 * (j + 1)
        a, c = f(x0) * sc, f(x1) * sc
        if float(f(x0)) == x0 and float(f(x1)) == x1 and c - a == f(8) and f(a + f(6)) >= c:
            found.append((x0, x1))
            if len(found) == count:
                return found
    return found


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("band", [25, 26])
@pytest.mark.parametrize("heads,tokens", [(4, 3), (64, 300), (64, 600), (64, 250)])
def test_a_largest_score_one_number_past_the_others(hip_ctx, heads, tokens, band, dtype):
    """All values of a head's dim are one number, so that any weights give that number."""
    rng = np.random.default_rng(band)
    hd, n = 64, tokens + 70
    pairs = large_scores(band, 40)
    assert len(pairs) == 40
    # x = 16384 a + 32 b + 32 c, all exact in f16 and in float32 sums: a the multiple of 16 that f16 holds
    k = np.zeros((n, heads, hd), np.float16)
    for h in range(heads):
        x0, x1 = pairs[h % 40]
        a = x0 // 16384 // 32 * 32
        rest = (x0 - 16384 * a) // 32
        high, low = divmod(rest, 1024)
        assert float(np.float16(a)) == a and high < 2048 and x0 == 16384 * a + 32768 * high + 32 * low
        k[:, h, 0], k[:, h, 1], k[:, h, 2] = a, high, low
        k[40:, h, 3] = (x1 - x0) // 32  # the larger score from the second step of 32 keys on
    q = np.zeros((tokens, heads, hd), NP[dtype])
    q[:, :, 0], q[:, :, 1], q[:, :, 2], q[:, :, 3] = 16384, 32768, 32, 32
    v = np.broadcast_to(rng.standard_normal((1, heads, hd)), (n, heads, hd)).astype(np.float16)
    b = Batch(rng, 16, [tokens], [n])
    cache = make(hip_ctx, b, heads, hd)
    with Device(hip_ctx) as dev:
        append(dev, cache, ref.whole(rng, b).on(dev), k, v, "f16")
        got = attend(dev, cache, b.on(dev), q, dtype)
    cache.close()
    want = v[:tokens].astype(np.float64)
    # the sums' half steps for each of n keys, the probabilities' (f16: one term, 2^-11; float32: two, 2^-22), the output's
    rel = (2 * n + 64) * 2.0 ** -24 + (2.0 ** -11 if dtype == "f16" else 2.0 ** -22)
    assert (np.abs(got - want) <= rel * np.abs(want) + ref.half_step(want, dtype)).all()
