"""Plain 64-bit forms of the operators over a KV cache in pages, and batches on
the device for their tests."""
import numpy as np

from alpaca_amd.kvcache import PagedBatch
from tests.q4_reference import EPS16, EPS32

NP = {"f32": np.float32, "f16": np.float16}


class Batch:
    """Sequences with `new` tokens of `lengths`; their pages drawn out of `pages` in a random order, but where
    `held`(s, page) says that a sequence has none (-1)."""

    def __init__(self, rng, page, new, lengths, pages=None, spare_rows=0, stride=None, held=None, lead=0):
        self.page, self.new, self.lengths, self.lead = page, list(new), list(lengths), lead
        self.starts = [lead + sum(new[:i]) for i in range(len(new) + 1)]
        self.rows = self.starts[-1] + spare_rows
        count = [-(-n // page) for n in lengths]
        self.stride = max(count + [1]) if stride is None else stride
        self.table = np.full((len(new), self.stride), -1, np.int32)
        want = [(s, p) for s, c in enumerate(count) for p in range(min(c, self.stride)) if held is None or held(s, p)]
        self.pages = len(want) + 2 if pages is None else pages
        for (s, p), i in zip(want, rng.permutation(self.pages)):
            self.table[s, p] = i

    def on(self, dev, hint=True):
        """The batch on the device, with or without its most rows."""
        a = [dev.put(np.array(x, np.int32)) for x in (self.starts, self.lengths, self.table)]
        return PagedBatch(*a, len(self.new), self.stride, self.rows, max(self.new + [0]) if hint else 0)

    def positions(self):
        """(sequence, position) of every row that has one."""
        return [(s, n - m + i) for s, (m, n) in enumerate(zip(self.new, self.lengths)) for i in range(m)]

    def sequence_rows(self, s):
        return slice(self.starts[s], self.starts[s + 1])


def whole(rng, batch):
    """The batch that writes every position of `batch`'s sequences, over the same pages."""
    b = Batch(rng, batch.page, batch.lengths, batch.lengths, batch.pages, stride=batch.stride)
    b.table = batch.table
    return b


def rotated(x, positions, table, interleaved):
    """Rows x [tokens, heads, hd] at their positions, in float64, and how far float32 arithmetic may be off: two products
    and their sum, half a step each of |a| + |b| at most (a fused one loses less)."""
    cos, sin = (table[positions][:, None, :, i].astype(np.float64) for i in range(2))
    x = x.astype(np.float64)
    hd = x.shape[-1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])

    def put(u, v):
        return np.stack([u, v], -1).reshape(x.shape) if interleaved else np.concatenate([u, v], -1)
    size = 3 * EPS32 * (np.abs(a) + np.abs(b))
    return put(a * cos - b * sin, a * sin + b * cos), put(size, size)


def half_step(x, dtype):
    """Of a value's rounding to the type."""
    return EPS32 * np.abs(x) + 2.0 ** -150 if dtype == "f32" else EPS16 * np.abs(x) + 2.0 ** -25


def sees(pos, length, window, sinks):
    """The positions that a query sees."""
    j = np.arange(min(max(pos + 1, 0), length))
    return j[(j > pos - window) | (j < sinks)] if window else j


def attention(q, k, v, first, dtype, window=0, sinks=0, heads=None):
    """Of queries q [tokens, heads, hd] at positions first.. over a sequence's keys and values [length, kv_heads, hd] as
    the cache holds them: float64, and how far the kernels' output may be off.

    A score: its hd products and their sums, the query's two f16 terms (2^-24 of its largest value each) and the
    scaling each lose at most half a float32 step of the sum of magnitudes; the probability as much as its
    score, and the exponential's 2^-22; numerator and denominator both.  The probabilities enter the products as two f16
    terms of p * 2^9, p against a reference that the row's largest is at least: past the terms' 2^-22 they are off by half
    of f16's smallest step, 2^-25 * 2^-9, each.  The sums over the keys lose a half step of the sum of magnitudes for
    every key.  In f16 queries, keys and values are exact; the probability in the numerator loses half an f16 step, and so
    does the output."""
    T, H, hd = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(H) if heads is None else heads:
        kh, vh = k[:, h // G].astype(np.float64), v[:, h // G].astype(np.float64)
        x = q[:, h].astype(np.float64)
        score, size = x @ kh.T / np.sqrt(hd), np.abs(x) @ np.abs(kh).T / np.sqrt(hd)
        for t in range(T):
            j = sees(first + t, len(k), window, sinks)
            n = len(j)
            if n == 0:
                continue
            p = np.exp(score[t, j] - score[t, j].max())
            p /= p.sum()
            out[t, h] = p @ vh[j]
            rel = 2 * ((hd + 16) * EPS32 * size[t, j].max() + 2.0 ** -22) + (n + 64) * EPS32
            small = n * 2.0 ** -34 * np.abs(vh[j]).max()
            if dtype == "f16":
                rel += EPS16
                small += EPS16 * np.abs(out[t, h]) + 2.0 ** -25
            bound[t, h] = rel * (p @ np.abs(vh[j])) + small
    return out, bound


def logprobs(x, tokens, top):
    """Of logits x [rows, vocab]: log probabilities of the tokens, entropies, top tokens with theirs, and bounds.

    A thread sums vocab / 256 terms at most one after the other, and as often moves its reference; 64 more steps join
    threads and parts: each a half step, and an exponential's 2^-22.  A difference to the maximum loses a half step of
    itself, the logarithm two; the sum of e^d d is of terms of magnitude e^d |d|."""
    x64 = x.astype(np.float64)
    rows, vocab = x64.shape
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x64.max(-1, keepdims=True)
        d = x64 - m
        e = np.exp(d)
        s = e.sum(-1, keepdims=True)
        ls = np.log(s)
        t = np.where(e == 0, 0, e * np.where(e == 0, 0, d)).sum(-1, keepdims=True) / s
        lp = d - ls
        # (a number before a NaN, larger ones first, then the lower index)
        order = [np.lexsort((np.arange(vocab), np.where(np.isnan(r), 0, -r), np.isnan(r)))[:top] for r in x64]
        best = np.array(order, np.int64).reshape(rows, top)
        sums = (vocab / 256 + 64) * EPS32 + 2.0 ** -22
        off = sums + 2 * EPS32 * np.abs(ls) + 2 * EPS32 * (np.abs(np.where(np.isfinite(d), d, 0)) + np.abs(ls))
        tok = np.clip(tokens, 0, vocab - 1)[:, None]
        one = np.take_along_axis(lp, tok, 1)[:, 0]
        one[(tokens < 0) | (tokens >= vocab)] = np.nan
        entropy = (ls - t)[:, 0]
        entropy_off = (2 * sums * (1 + np.abs(t)) + 4 * EPS32 * (np.abs(ls) + np.abs(t)))[:, 0]
    return (one, entropy, best, np.take_along_axis(lp, best, 1),
            (np.take_along_axis(off, tok, 1)[:, 0], entropy_off, np.take_along_axis(off, best, 1)))
