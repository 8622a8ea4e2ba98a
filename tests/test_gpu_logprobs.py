"""Log probabilities, entropies and top tokens on the GPU against 64-bit plain forms."""
import ctypes as C

import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd import synth
from alpaca_amd.model import HIPLlamaModel
from alpaca_amd.sampling import LOGPROBS_WORKSPACE_ZERO, token_logprobs
from tests import paged_reference as ref
from tests.paged_reference import NP
from tests.q4_reference import Device

pytestmark = pytest.mark.gpu


def run(ctx, x, tokens, top, extra=0, lead=0, **kw):
    """x [rows, vocab] as it lies `extra` elements apart and `lead` from where it could."""
    n, vocab = x.shape
    stride = vocab + extra
    flat = np.full(lead + n * stride, 1000, x.dtype)
    flat[lead:].reshape(n, stride)[:, :vocab] = x
    with Device(ctx) as dev:
        lp, en, tt, tl = (dev.empty(max(4 * n * m, 1)) for m in (1, 1, top, top))
        token_logprobs(ctx, dev.put(flat) + lead * x.itemsize, n, vocab, dev.put(tokens.astype(np.int32)), lp, en, top, tt,
                       tl, "f16" if x.dtype == np.float16 else "f32", stride, **kw)
        return (dev.get(lp, n, np.float32), dev.get(en, n, np.float32), dev.get(tt, (n, top), np.int32),
                dev.get(tl, (n, top), np.float32))


def equal_or_near(got, want, bound):
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        return (same | (np.abs(got - want) <= bound)).all()


def check(ctx, x, tokens, top, **kw):
    one, entropy, best, tops, (a, b, c) = ref.logprobs(x, tokens, top)
    got = run(ctx, x, tokens, top, **kw)
    assert np.array_equal(got[2], best)
    assert equal_or_near(got[0], one, a) and equal_or_near(got[1], entropy, b) and equal_or_near(got[3], tops, c)
    return got


def some(rng, rows, vocab, dtype, size=2.5):
    x = (rng.standard_normal((rows, vocab)) * size).astype(NP[dtype])
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 9
    return x, rng.integers(0, vocab, rows)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 3, 3), (5, 7, 0), (2, 32, 32), (3, 33, 32), (4, 255, 5), (1, 1025, 1),
                                            (7, 4097, 20), (1, 49152, 5), (3, 49152, 32), (40, 30001, 12), (1, 150001, 32),
                                            (600, 5003, 8), (513, 2048, 1), (512, 8200, 3)])
def test_rows_of_every_size(hip_ctx, rows, vocab, top, dtype):
    rng = np.random.default_rng(rows * 7 + vocab)
    x, tokens = some(rng, rows, vocab, dtype)
    check(hip_ctx, x, tokens, top)
    if rows <= 40:
        check(hip_ctx, x, tokens, top, extra=5, lead=3)


@pytest.mark.parametrize("rows", [1, 300])
def test_a_workspace_changes_rounding_only(hip_ctx, rows):
    rng = np.random.default_rng(rows)
    x, tokens = some(rng, rows, 20000, "f32")
    split = check(hip_ctx, x, tokens, 9)
    with Device(hip_ctx) as dev:
        n = C.c_int64()
        L.check(L.lib().ahip_token_logprobs_workspace(C.byref(n)))
        mine = dev.empty(n.value, 0xFF)  # its bytes NaN but for the counters
        L.check(L.lib().ahip_memset(hip_ctx.handle, mine, 0, LOGPROBS_WORKSPACE_ZERO))
        again = run(hip_ctx, x, tokens, 9, workspace=(mine, n.value))
        assert not dev.get(mine, LOGPROBS_WORKSPACE_ZERO, np.uint8).any()
    assert all(np.array_equal(a.view(np.uint8), b.view(np.uint8)) for a, b in zip(split, again))
    check(hip_ctx, x, tokens, 9, workspace=(None, 0))  # a row a workgroup


# rows that are hard to rank, and rows that hold more than numbers
def ascending(n):
    return np.linspace(-5, 5, n)


def one_group(n):
    """The largest values all where one group of threads reads (the groups of 64 share 1,024 elements f32)."""
    x = np.linspace(-5, -4, n)
    mine = (np.arange(n) % 1024) // 16 == 5
    x[mine] = np.linspace(3, 4, mine.sum())
    return x


def one_group_f16(n):
    x = np.linspace(-5, -4, n)
    mine = (np.arange(n) % 2048) // 32 == 5
    x[mine] = np.linspace(3, 4, mine.sum())
    return x


def masked(n):
    """Ten tokens that are allowed."""
    x = np.full(n, -np.inf)
    x[np.linspace(0, n - 1, 10).astype(int)] = np.arange(10) % 4
    return x


def masked_at_first(n):
    x = np.full(n, -np.inf)
    x[n // 2:] = 0.5
    return x


def with_value(value, at):
    def f(n):
        x = np.sin(np.arange(n) * 0.37)
        x[at if at >= 0 else n + at] = value
        return x
    return f


def mostly_nan(n):
    x = np.full(n, np.nan)
    x[[3, n // 2, n - 1]] = 1, 2, -np.inf
    return x


ROWS = [ascending, lambda n: ascending(n)[::-1].copy(), one_group, one_group_f16, lambda n: np.zeros(n),
        lambda n: np.arange(n) % 3 + 0.0, lambda n: -(np.arange(n) // 500 % 2 + 0.0), masked, masked_at_first,
        lambda n: np.full(n, -np.inf), lambda n: np.full(n, np.nan), mostly_nan, with_value(np.nan, 0), with_value(np.nan, -1),
        with_value(np.inf, 5), with_value(-np.inf, 5), with_value(6e4, -3), lambda n: np.full(n, 6e4),
        lambda n: np.where(np.arange(n) % 2, 0.0, -0.0), lambda n: np.arange(n) * -1e3 / n * 60]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [40, 3001, 100000])
@pytest.mark.parametrize("top", [2, 20, 32])
def test_rows_that_are_hard_to_rank(hip_ctx, vocab, top, dtype):
    for i, make in enumerate(ROWS):
        x = make(vocab).astype(NP[dtype])[None]
        for tokens in ([0], [vocab - 1], [-1], [vocab]):
            for kw in ({}, {"workspace": (None, 0)}) if tokens == [0] else ({},):
                try:
                    check(hip_ctx, x, np.array(tokens), top, **kw)
                except AssertionError as e:
                    raise AssertionError(f"row {i} of {vocab}, {tokens}, {kw}") from e


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_hard_rows_at_once(hip_ctx, dtype):
    x = np.stack([make(7000) for make in ROWS] * 40).astype(NP[dtype])
    check(hip_ctx, x, np.arange(len(x)) * 7 % 7000, 10, extra=3)


def test_outputs_that_are_not_asked_for(hip_ctx):
    rng = np.random.default_rng(3)
    x, tokens = some(rng, 4, 3000, "f32")
    one, entropy, best, tops, (a, b, c) = ref.logprobs(x, tokens, 4)
    with Device(hip_ctx) as dev:
        lp, en, tt, tl = dev.empty(16), dev.empty(16), dev.empty(64), dev.empty(64)
        xp = dev.put(x)
        token_logprobs(hip_ctx, xp, 4, 3000, entropy=en)
        token_logprobs(hip_ctx, xp, 4, 3000, tokens=dev.put(tokens.astype(np.int32)), logprobs=lp)
        token_logprobs(hip_ctx, xp, 4, 3000, top=4, top_tokens=tt, top_logprobs=tl)
        assert equal_or_near(dev.get(en, 4, np.float32), entropy, b) and equal_or_near(dev.get(lp, 4, np.float32), one, a)
        assert np.array_equal(dev.get(tt, (4, 4), np.int32), best)
        assert equal_or_near(dev.get(tl, (4, 4), np.float32), tops, c)


def test_a_session_s_logits(hip_ctx):
    spec = synth.TINY
    model = HIPLlamaModel(hip_ctx, spec.config, synth.build_weights(spec))
    s = model.make_session(capacity=64)
    with pytest.raises(L.InvalidArgument, match="no logits"):
        s.logprobs(0)
    for step in range(3):
        logits = s.forward(synth.prompt_tokens(spec, 9)) if step == 0 else s.decode(token)
        logits = np.array(logits, np.float32)[None]
        token = s.sample(0.9, 40, 0.95, 0.3 + 0.2 * step)
        one, entropy, best, tops, (a, b, c) = ref.logprobs(logits, np.array([token]), 6)
        lp, en, top = s.logprobs(token, 6)
        assert abs(lp - one[0]) <= a[0] and abs(en - entropy[0]) <= b[0]
        assert [t for t, _ in top] == best[0].tolist() and equal_or_near(np.array([[x for _, x in top]]), tops, c)
        assert s.logprobs(token) == (lp, en, [])
        assert s.sample(0.0) == best[0, 0]  # (the logits are still there)
    for bad in (-1, spec.config.vocab_size):
        with pytest.raises(L.InvalidArgument, match="outside vocabulary"):
            s.logprobs(bad)
    for bad in (-1, 33):
        with pytest.raises(L.InvalidArgument, match="top"):
            s.logprobs(0, bad)
    s.reset()
    with pytest.raises(L.InvalidArgument, match="no logits"):
        s.logprobs(0)
    s.close()
    model.close()
