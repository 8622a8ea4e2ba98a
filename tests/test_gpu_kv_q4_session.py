"""Sessions with a KV cache in 4 bits, and the op-level calls over one, against
a 64-bit forward pass whose keys and values go through the quantiser."""
import numpy as np
import pytest

import oracle.oracle as orc
from alpaca_amd import _lib as L
from alpaca_amd import synth
from alpaca_amd.model import HIPLlamaModel
from alpaca_amd.ops import HIPOps
from alpaca_amd.tensor import F16, F32, Q4_0
from tests import q4_reference as ref

pytestmark = pytest.mark.gpu

_models = {}


def gpu_model(ctx, spec):
    if spec.name not in _models:
        w = synth.build_weights(spec)
        _models[spec.name] = (HIPLlamaModel(ctx, spec.config, w), w)
    return _models[spec.name]


class Forward:
    """Llama in float64 over the stored weights, the cache in 4 bits; `flip`: values of the cache within `near` of a
    border of the quantiser go to its other side."""

    def __init__(self, config, weights, flip=False, near=2e-4):
        self.c, self.flip, self.near = config, flip, near
        self.w = {n: (t.data.view(np.float32) if t.dtype == F32 else
                      orc.dequantize(t.dtype, t.data, t.rows * t.cols)).astype(np.float64).reshape(t.rows, t.cols)
                  for n, t in weights.items()}
        self.kv = [[None, None] for _ in range(config.layer_count)]
        self.n = 0

    def quantised(self, x):
        x = x.astype(np.float32)
        y = ref.q4_values(x)
        if self.flip:
            b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
            d = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1) / -8
            s = np.where(d != 0, b / np.where(d == 0, 1, d), 0) + 8.5
            border = np.round(s)
            other = np.where(np.abs(s - border) < self.near, np.where(s >= border, border - 1, border), np.trunc(s))
            y = (d.astype(np.float16).astype(np.float64) * (other.clip(0, 15) - 8)).reshape(x.shape)
        return y

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.rms_norm_eps) * w

    def __call__(self, tokens):
        c, w, T, hd = self.c, self.w, len(tokens), self.c.head_dim
        x = w["token_embd"][np.asarray(tokens)]
        angle = (self.n + np.arange(T))[:, None] * c.rope_theta ** (-2.0 * np.arange(hd // 2) / hd)
        cs = np.stack([np.cos(angle), np.sin(angle)], -1)
        for li in range(c.layer_count):
            m = {n: w[f"blk.{li}.{n}"] for n in synth.LAYER_TENSORS}
            h = self.norm(x, m["attn_norm"])
            q = ref.norm_rope((h @ m["attn_q"].T).reshape(T, -1, hd), None, 0, cs, True)
            k = ref.norm_rope((h @ m["attn_k"].T).reshape(T, -1, hd), None, 0, cs, True)
            new = self.quantised(k), self.quantised((h @ m["attn_v"].T).reshape(T, -1, hd))
            for i in (0, 1):
                old = self.kv[li][i]
                self.kv[li][i] = new[i] if old is None else np.concatenate([old, new[i]])
            o, _ = ref.attention(q, *self.kv[li], self.n, "f32")
            x = x + o.reshape(T, -1) @ m["attn_output"].T
            h = self.norm(x, m["ffn_norm"])
            g = h @ m["ffn_gate"].T
            x = x + (g / (1 + np.exp(-g)) * (h @ m["ffn_up"].T)) @ m["ffn_down"].T
        self.n += T
        return (self.norm(x[-1:], w["output_norm"]) @ w.get("output", w["token_embd"]).T)[0]


def check(got, ref_a, ref_b, prec, label):
    """The logits' bar of the library's float32 and two-term modes (2e-3 + 1e-3 relative), or of one f16 term (3e-3 of
    the peak), and past it what values on a border of the quantiser can move: they may fall on either side."""
    bar = 2e-3 + 1e-3 * np.abs(ref_a) if prec != "fast-f16" else 3e-3 * np.abs(ref_a).max() + 1e-3 * np.abs(ref_a)
    bound = bar + 2 * np.abs(ref_a - ref_b).max()
    off = np.abs(got - ref_a)
    print(f"[logits] {label}: max |d| {off.max():.2e}, borders {np.abs(ref_a - ref_b).max():.2e}, "
          f"{(off / bound).max():.3f} of the bound")
    assert (off <= bound).all(), label


@pytest.mark.parametrize("spec", [synth.TINY, synth.with_dtype(synth.TINY, Q4_0), synth.with_dtype(synth.TINY, F16)],
                         ids=lambda s: s.name)
@pytest.mark.parametrize("prec", ["exact", "fast", "fast-f16"])
def test_session_matches_the_quantised_forward(hip_ctx, spec, prec):
    """A prompt, a second message, a short one of a few tokens and single tokens."""
    model, w = gpu_model(hip_ctx, spec)
    # in steps of the quantiser, 8 to a block's largest value: a sum of 512 float32 products is off by some
    # sqrt(512) 2^-24 of its magnitudes, themselves several times a value, in each of three layers; one f16 term
    # moves a value by up to 2^-11
    near = 2e-4 if prec != "fast-f16" else 2e-2
    a, b = Forward(spec.config, w), Forward(spec.config, w, True, near)
    s = model.make_session(capacity=160, max_batch=64, kv_precision="q4_0", gemm_precision=prec)
    prompt = synth.prompt_tokens(spec, 110)
    for part in (prompt[:40], prompt[40:75], prompt[75:82], prompt[82:83], prompt[83:84], prompt[84:]):
        got = s.forward(part)
        check(got, a(part), b(part), prec, f"{spec.name} {prec} {len(part)} tokens at {s.length - len(part)}")
    assert s.length == 110


@pytest.mark.parametrize("prec", ["exact", "fast"])
def test_greedy_chain_replays_the_decoded_steps(hip_ctx, prec):
    """The captured graph, replayed with other work and waits between, gives the tokens of single decode calls."""
    model, _ = gpu_model(hip_ctx, synth.TINY)
    prompt = synth.prompt_tokens(synth.TINY, 37)
    one = model.make_session(capacity=128, kv_precision="q4_0", gemm_precision=prec)
    token = int(np.argmax(one.forward(prompt)))
    first, want = token, []
    for _ in range(60):
        token = int(np.argmax(one.decode(token)))
        want.append(token)
    for profiled in (False, True, False):
        s = model.make_session(capacity=128, kv_precision="q4_0", gemm_precision=prec)
        s.profiling_enabled = profiled
        assert int(np.argmax(s.forward(prompt))) == first
        got = []
        for n in (20, 1, 39):  # three chains, replays of one graph
            s.decode_greedy(got[-1] if got else first, n, lambda t: got.append(t) or True)
            other = model.make_session(capacity=64)
            other.forward(prompt[:20])
            other.close()
        assert got == want
        if profiled:
            assert s.last_profile["attention"].dispatches == 39 * synth.TINY.config.layer_count


def test_two_sessions_at_once_and_reset(hip_ctx):
    model, _ = gpu_model(hip_ctx, synth.TINY)
    prompt = synth.prompt_tokens(synth.TINY, 90)
    a = model.make_session(capacity=128, kv_precision="q4_0")
    b = model.make_session(capacity=1024, kv_precision="q4_0")
    first = a.forward(prompt)
    other = b.forward(prompt[::-1])
    a.reset()
    assert np.array_equal(a.forward(prompt), first)
    b.reset()
    assert np.array_equal(b.forward(prompt[::-1]), other)
    assert not np.array_equal(first, other)


def test_chunked_prompt_is_the_prompt(hip_ctx):
    """In exact mode a row's arithmetic does not depend on its chunk, so the caches and the logits are equal."""
    model, _ = gpu_model(hip_ctx, synth.TINY)
    prompt = synth.prompt_tokens(synth.TINY, 120)
    out = []
    for batch in (512, 120, 40):
        s = model.make_session(capacity=128, max_batch=batch, kv_precision="q4_0", gemm_precision="exact")
        out.append(s.forward(prompt))
    assert np.array_equal(out[0], out[1])
    assert np.abs(out[0] - out[2]).max() <= 2e-3 + 1e-3 * np.abs(out[0]).max()


def test_split_prefill_with_a_4_bit_cache(hip_ctx, monkeypatch):
    """A prompt whose halves run on two streams, its middle inside a tile of the cache."""
    model, w = gpu_model(hip_ctx, synth.TINY)
    prompt = synth.prompt_tokens(synth.TINY, 700)
    out = []
    for least in ("100000", "512"):
        monkeypatch.setenv("ALPACA_HIP_SPLIT_MIN", least)
        s = model.make_session(capacity=1024, max_batch=1024, kv_precision="q4_0", gemm_precision="fast-f16")
        s.forward(prompt[:13])
        out.append(s.forward(prompt[13:]))
    peak = np.abs(out[0]).max()
    assert np.isfinite(out[1]).all() and np.abs(out[0] - out[1]).max() <= 0.05 * peak


def test_session_bytes_and_refusals(hip_ctx):
    c = synth.C1.config
    f16 = HIPLlamaModel.session_byte_count(c, 2048, 512, "f16")
    q4 = HIPLlamaModel.session_byte_count(c, 2048, 512, "q4_0")
    cache = 2 * c.layer_count * 2048 * c.kv_width
    assert cache * 18 // 32 < q4 - (f16 - 2 * cache) < cache * 18 // 32 + (64 << 20)  # the cache and its workspaces
    model, _ = gpu_model(hip_ctx, synth.TINY)
    s = model.make_session(capacity=32, kv_precision="q4_0")
    with pytest.raises(L.InvalidArgument):
        s.forward(np.zeros(33, np.int32))
    s.forward(np.zeros(32, np.int32))
    with pytest.raises(L.InvalidArgument):
        s.decode(1)
    assert s.length == 32


@pytest.mark.parametrize("prec", ["exact", "fast", "fast-f16"])
@pytest.mark.parametrize("tokens,start,heads,kv_heads,hd", [(1, 0, 4, 2, 64), (1, 300, 6, 3, 128), (20, 13, 6, 2, 96),
                                                            (70, 40, 9, 3, 64), (33, 0, 2, 1, 256)])
def test_op_attention(hip_ctx, prec, tokens, start, heads, kv_heads, hd):
    rng = np.random.default_rng(tokens + hd)
    q = rng.standard_normal((tokens, heads, hd)).astype(np.float32)
    k, v = (rng.standard_normal((start + tokens + 5, kv_heads, hd)).astype(np.float32) for _ in range(2))
    got = HIPOps(hip_ctx).attention(q, k, v, start, "q4_0", prec)
    half = prec == "fast-f16" and tokens >= 16
    if half:
        q = q.astype(np.float16)
    kd, vd = ref.q4_rows(k, v)
    n = start + tokens
    want, bound = ref.attention(q, kd[:n], vd[:n], start, "f16" if half else "f32")
    assert (np.abs(got - want) <= bound).all()


def test_op_qk_norm_rope(hip_ctx):
    ops = HIPOps(hip_ctx)
    rng = np.random.default_rng(8)
    q, k = (rng.standard_normal((5, n, 64)).astype(np.float32) for n in (6, 2))
    gq, gk = ((1 + 0.1 * rng.standard_normal(64)).astype(np.float32) for _ in range(2))
    angle = (7 + np.arange(5))[:, None] * 1e4 ** (-2.0 * np.arange(32) / 64)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1)
    for inter in (True, False):
        got = ops.qk_norm_rope(q, k, 7, 1e4, gq, gk, 1e-6, inter)
        for g, x, gain in zip(got, (q, k), (gq, gk)):
            # the norm's hd / 2 + 6 half steps, the rotation's and the table's, of values below sqrt(64) * 1.5
            assert np.abs(g - ref.norm_rope(x, gain, 1e-6, cs, inter)).max() <= 48 * ref.EPS32 * 12
    # no gain: the rotation alone, as HIPOps.rope gives it
    got = ops.qk_norm_rope(q, k, 7, 1e4)
    assert np.abs(got[0] - ops.rope(q, 7, 1e4)).max() <= 3 * ref.EPS32 * np.abs(q).max() * 2
    with pytest.raises(L.InvalidArgument):
        ops.qk_norm_rope(q, k[:4], 0, 1e4)
    with pytest.raises(L.InvalidArgument):
        ops.qk_norm_rope(q, k, 0, 1e4, gq[:32])
    with pytest.raises(L.InvalidArgument):
        ops.qk_norm_rope(q[..., :48], k[..., :48], 0, 1e4)
