"""Plain 64-bit forms of the operators around the 4-bit KV cache, and device
buffers for their tests."""
import ctypes as C

import numpy as np

from alpaca_amd import _lib as L

EPS32, EPS16 = 2.0 ** -24, 2.0 ** -11  # half a step of float32 and f16, relative


class Device:
    """Arrays on the device, freed together."""

    def __init__(self, ctx):
        self.ctx, self.held = ctx.handle, []

    def __enter__(self):
        return self

    def __exit__(self, *_):
        for p in self.held:
            L.lib().ahip_free(self.ctx, p)

    def empty(self, nbytes, fill=0xA5):
        """Bytes of `fill`."""
        p = C.c_void_p()
        L.check(L.lib().ahip_malloc(self.ctx, nbytes, C.byref(p)))
        self.held.append(p.value)
        L.check(L.lib().ahip_memset(self.ctx, p, fill, nbytes))
        return p.value

    def put(self, a):
        a = np.ascontiguousarray(a)
        p = self.empty(max(a.nbytes, 1))
        if a.nbytes:
            L.check(L.lib().ahip_memcpy_htod(self.ctx, p, a.ctypes.data, a.nbytes))
        return p

    def get(self, p, shape, dtype):
        a = np.empty(shape, dtype)
        if a.nbytes:
            L.check(L.lib().ahip_memcpy_dtoh(self.ctx, a.ctypes.data, p, a.nbytes))
        return a


def q4_values(x):
    """What float32 rows [..., hd] read back as (float64), where they have a form.

    The float32 steps of the format, each exact in float64 and then rounded."""
    b = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    at = np.abs(b).argmax(-1)[..., None]  # the first of equal magnitudes
    d = np.take_along_axis(b, at, -1) / -8
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(d != 0, np.float32(1) / d.astype(np.float32), np.float32(0)).astype(np.float64)
        n = np.trunc((((b * inv).astype(np.float32)) + np.float32(8.5)).astype(np.float64)).clip(0, 15)
        d = d.astype(np.float16).astype(np.float64)
        # (a scale that f16 rounds to zero: whatever nibble 1 / d gave, zeros)
        return np.where(d == 0, 0, d * (n - 8)).reshape(x.shape)


def q4_rows(k, v):
    """(keys, values) [tokens, kv_heads, hd] as they read back: NaN where a token's head has no form."""
    odd = ~((np.abs(k) <= 65504).all(-1) & (np.abs(v) <= 65504).all(-1))
    out = []
    for x in (k, v):
        y = q4_values(np.where(odd[..., None], 0, x).astype(np.float32))
        y[odd] = np.nan
        out.append(y)
    return out


def attention(q, k, v, start, dtype):
    """Causal attention in float64, and how far the kernels' output may be from it.

    q [tokens, heads, hd], k and v [length, kv_heads, hd].  A score: its hd products and their sums, the query's
    two f16 terms (2^-24 of its largest value each) and the scaling each lose at most half a float32 step of the sum
    of magnitudes; the probability as much as its score, and the exponential's 2^-22; numerator and denominator
    both.  The probabilities enter the products as two f16 terms of p * 2^14, p against the largest of the row: past
    the terms' 2^-22 they are off by half of f16's smallest step, 2^-25 * 2^-14, each.  The sums over the keys lose
    a half step of the sum of magnitudes for every key.  In f16 the keys are exact; the probability (of numerator and
    denominator) and the value each lose half an f16 step, and so does the output."""
    T, H, hd = q.shape
    G = H // k.shape[1]
    out, bound = np.empty(q.shape), np.empty(q.shape)
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        for t in range(T):
            n, x = start + t + 1, q[t, h].astype(np.float64)
            s = kh[:n] @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vh[:n]
            size = (np.abs(kh[:n]) @ np.abs(x)).max() / np.sqrt(hd)
            rel = 2 * ((hd + 16) * EPS32 * size + 2.0 ** -22) + (n + 64) * EPS32
            small = n * 2.0 ** -39 * np.abs(vh[:n]).max()
            if dtype == "f16":
                rel, small = rel + 3 * EPS16, small + EPS16 * np.abs(out[t, h]) + 2.0 ** -24
            bound[t, h] = rel * (p @ np.abs(vh[:n])) + small
    return out, bound


def norm_rope(x, gain, eps, cs, interleaved):
    """x [tokens, heads, hd]; cs [tokens, hd / 2, 2] or None; float64."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    if cs is None:
        return x
    hd = x.shape[-1]
    cos, sin = cs[:, None, :, 0].astype(np.float64), cs[:, None, :, 1].astype(np.float64)
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return np.stack([a, b], -1).reshape(x.shape) if interleaved else np.concatenate([a, b], -1)
