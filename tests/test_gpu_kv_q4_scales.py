"""Attention over the 4-bit KV cache where the values of the tokens differ
widely in size: what a query gives no weight to must not cost the others'
accuracy."""
import numpy as np
import pytest

from alpaca_amd.kvcache import Q4Cache
from tests import q4_reference as ref
from tests.test_gpu_kv_q4 import NP, run_attention, store

pytestmark = pytest.mark.gpu

L2E = 1.4427


def single_tokens(q, k, v, start, dtype):
    """Attention in float64 of the calls with few query columns, and how far the kernel may be from it.

    A probability p_k is off, relatively, by its score's hd products and sums and the query's two terms (half a float32
    step of the sum of magnitudes each), by the exponential's argument (base 2: its own rounding and that of what is
    taken out of it, the maximum and an exponent with 14 below 40; 2 ln 2 < 1.5 half steps) and by 2^-22 for the
    exponential and for each of up to 8 rescalings; numerator and denominator both.  The sums lose half a step of the
    sum of magnitudes a key.  The products of p_k and its value's scale d_k enter as two f16 terms: past their 2^-22,
    half of f16's smallest step, 2^-25, where the largest of the block's products so far is at 2^13 or more; times a
    quant, at most 8."""
    T, H, hd = q.shape
    G = H // k.shape[1]
    out, bound = np.empty(q.shape), np.empty(q.shape)
    for t in range(T):
        for h in range(H):
            n, x = start + t + 1, q[t, h].astype(np.float64)
            kh, vh = k[:n, h // G], v[:n, h // G]
            s = kh @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vh
            size = np.abs(x).max() * np.abs(kh).sum(-1) / np.sqrt(hd)
            rel = ((hd + 16) * size + 1.5 * (L2E * (s.max() - s + abs(s.max())) + 40)) * ref.EPS32 + 10 * 2.0 ** -22
            if dtype == "f16":
                rel = rel + 2 * ref.EPS16  # the probability times the scale, one f16 term
            d = np.abs(vh).reshape(n, -1, 32).max(-1) / 7  # (a block's largest quant is 8 or 7)
            small = np.repeat(n * 2.0 ** -38 * 8 * (p[:, None] * d).max(0), 32)
            bound[t, h] = ((p * rel) @ np.abs(vh) + np.abs(out[t, h]) * (p @ rel) +
                           (n + 64) * ref.EPS32 * (p @ np.abs(vh)) + small)
            if dtype == "f16":
                bound[t, h] += ref.EPS16 * np.abs(out[t, h]) + 2.0 ** -25
    return out, bound


# (heads, kv_heads, head_dim, tokens, positions before them)
SHAPES = [(1, 1, 64, 1, 299), (8, 2, 64, 1, 300), (4, 1, 64, 2, 333), (16, 1, 32, 1, 500), (3, 1, 96, 1, 2000),
          (4, 1, 128, 1, 270), (8, 2, 128, 1, 6000), (2, 1, 160, 1, 400), (2, 1, 256, 1, 1100)]


def case(rng, kind, size, n, hd, kv_heads):
    """Scores (for a query of ones) and values [n, kv_heads, hd]."""
    s = rng.standard_normal((n, kv_heads)) * 0.5
    v = rng.standard_normal((n, kv_heads, hd)) * size
    if kind.startswith("outlier"):  # values of 60,000 at a weight of e^-60
        at = {"first": 0, "middle": n // 2, "last": n - 3}[kind[8:]]
        s[at], v[at] = -60, 6e4 * np.sign(rng.standard_normal((kv_heads, hd)))
    elif kind == "rising":  # the outlier has the largest score of its part of the keys, until later ones come
        s[:n // 2] -= 60
        s[3], v[3] = -58, 6e4
    elif kind == "sink":  # nearly all weight on a token of almost no value
        s[1:] -= 14
        s[0], v[0] = 2, 1e-6
    return s, v


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("size", [1e-5, 1e-3, 1.0])
@pytest.mark.parametrize("kind", ["outlier first", "outlier middle", "outlier last", "rising", "sink"])
@pytest.mark.parametrize("heads,kv_heads,hd,tokens,start", SHAPES)
def test_single_tokens_keep_their_accuracy(hip_ctx, heads, kv_heads, hd, tokens, start, kind, size, dtype):
    rng = np.random.default_rng(heads * 1009 + hd * 31 + start)
    n = start + tokens
    s, v = case(rng, kind, size, n, hd, kv_heads)
    k = (s[..., None] / np.sqrt(hd) + 0.1 * rng.standard_normal((n, kv_heads, hd))).astype(np.float32)
    v = v.astype(np.float32)
    q = (1 + 0.05 * rng.standard_normal((tokens, heads, hd))).astype(NP[dtype])
    cache = Q4Cache(hip_ctx, kv_heads, n, hd)
    with ref.Device(hip_ctx) as dev:
        store(dev, cache, k, v, 0, "f32")
        got = run_attention(dev, cache, q, start, dtype).astype(np.float64)
    cache.close()
    want, bound = single_tokens(q, *ref.q4_rows(k, v), start, dtype)
    off = np.abs(got - want)
    print(f"[attention] {kind} {size} {dtype}: {(off / bound).max():.3f} of the bound, "
          f"{off.max() / np.abs(want).max():.2e} of the largest output")
    assert (off <= bound).all()
