"""Sessions with a KV cache in 4 bits, on a model whose keys and values stay
clear of the quantiser's borders: the logits are held to the library's bars
alone, which a forward pass of other cached values misses."""
import functools

import numpy as np
import pytest

from alpaca_amd import synth
from alpaca_amd.model import HIPLlamaModel, LlamaConfig
from alpaca_amd.tensor import F16, F32, Q4_0, Q8_0, encode
from tests.test_gpu_kv_q4_session import Forward

pytestmark = pytest.mark.gpu

THETA, CLEAR = 1e5, 0.1


@functools.cache
def build(heads, kv_heads, hd, layers, tokens, dtype):
    """(config, weights, prompt): the part of the residual stream that the layers' keys and values are taken from is
    written by the embedding alone, and a token stands at one position only.  A norm scales a token's row as a whole,
    so that where its values lie between two steps of their block does not depend on what the layers add to the rest.
    In steps, a block has one value of -8 or 8 and others in (-7.5, 7.5), CLEAR or more from a border (a half)."""
    rng = np.random.default_rng(heads * 100 + hd + layers)
    KW, QW, work = kv_heads * hd, heads * hd, 128
    H = 2 * KW + work
    c = LlamaConfig(vocab_size=tokens, hidden_size=H, layer_count=layers, head_count=heads, kv_head_count=kv_heads,
                    head_dim=hd, feed_forward_size=256, context_length=tokens + 32, rms_norm_eps=1e-5, rope_theta=THETA)

    def rows():
        r = rng.integers(-7, 8, (tokens, KW // 32, 32)) + rng.uniform(-0.5 + CLEAR, 0.5 - CLEAR, (tokens, KW // 32, 32))
        at = rng.integers(0, 32, (tokens, KW // 32, 1))
        np.put_along_axis(r, at, rng.choice([-8.0, 8.0], at.shape), -1)
        return r.reshape(tokens, KW)
    # the keys are rotated after their projection: back by the position's angle before it
    angle = np.arange(tokens)[:, None] * THETA ** (-2.0 * np.arange(hd // 2) / hd)
    k = rows().reshape(tokens, kv_heads, hd // 2, 2)
    co, si = np.cos(angle)[:, None], np.sin(angle)[:, None]
    k = np.stack([k[..., 0] * co + k[..., 1] * si, k[..., 1] * co - k[..., 0] * si], -1).reshape(tokens, KW)
    prompt = rng.permutation(tokens).astype(np.int32)
    embed = np.empty((tokens, H), np.float32)
    embed[prompt] = np.concatenate([k, rows(), 4 * rng.standard_normal((tokens, work))], 1)

    def random(r, cols, std=0.1):
        return (rng.standard_normal((r, cols)) * std).astype(np.float32)

    def added(cols, std):  # into the rest of the stream only
        return np.concatenate([np.zeros((2 * KW, cols), np.float32), random(work, cols, std)])
    w = {"token_embd": encode(embed, F16)}
    for li in range(layers):
        # a layer's own order of the heads, and of the values in a block
        k_from = np.concatenate([np.arange(hd) + hd * h for h in rng.permutation(kv_heads)])
        v_from = np.concatenate([rng.permutation(32) + 32 * b for b in rng.permutation(KW // 32)]) + KW
        one_k, one_v = np.zeros((KW, H), np.float32), np.zeros((KW, H), np.float32)
        one_k[np.arange(KW), k_from] = 1
        one_v[np.arange(KW), v_from] = rng.choice([-1, 1], KW // 32).repeat(32)
        m = {"attn_q": random(QW, H), "attn_k": one_k, "attn_v": one_v, "attn_output": added(QW, 0.4),
             "ffn_gate": random(256, H), "ffn_up": random(256, H), "ffn_down": added(256, 0.1)}
        for n in ("attn_norm", "ffn_norm"):
            w[f"blk.{li}.{n}"] = encode(np.ones((1, H), np.float32), F32)
        for n, x in m.items():
            w[f"blk.{li}.{n}"] = encode(x, dtype)
    w["output_norm"] = encode(np.ones((1, H), np.float32), F32)
    w["output"] = encode(np.concatenate([np.zeros((tokens, 2 * KW), np.float32), random(tokens, work)], 1), dtype)
    return c, w, prompt


class Other(Forward):
    """A forward pass whose cache holds other values."""

    def __init__(self, config, weights, change):
        super().__init__(config, weights)
        self.change = change

    def quantised(self, x):
        return self.change(x.astype(np.float32), super().quantised(x))


OTHERS = {"not quantised": lambda x, y: x.astype(np.float64), "3% larger": lambda x, y: 1.03 * y}


@functools.cache
def references(parts, *model):
    """The logits of every call, those with any value near a border on its other side, and those of OTHERS."""
    c, w, prompt = build(*model)
    passes = {"": Forward(c, w), "borders": Forward(c, w, True, CLEAR / 2)}
    passes.update((name, Other(c, w, change)) for name, change in OTHERS.items())
    out, at = [], 0
    for n in parts:
        out.append({name: f(prompt[at:at + n]) for name, f in passes.items()})
        at += n
    return out


def check(hip_ctx, parts, prec, *model):
    c, w, prompt = build(*model)
    m = HIPLlamaModel(hip_ctx, c, w)
    s = m.make_session(capacity=c.context_length, max_batch=512, kv_precision="q4_0", gemm_precision=prec)
    at = 0
    for n, want in zip(parts, references(parts, *model)):
        got, ref = s.forward(prompt[at:at + n]), want[""]
        assert np.array_equal(ref, want["borders"])  # no value lies near one
        bar = 2e-3 + 1e-3 * np.abs(ref) if prec != "fast-f16" else 3e-3 * np.abs(ref).max() + 1e-3 * np.abs(ref)
        off = {name: (np.abs(x - ref) / bar).max() for name, x in want.items() if name in OTHERS}
        print(f"[logits] {prec} {n} tokens at {at}: {(np.abs(got - ref) / bar).max():.3f} of the bar; "
              + ", ".join(f"{k} {v:.1f}" for k, v in off.items()))
        assert (np.abs(got - ref) <= bar).all(), (n, at)
        assert min(off.values()) > 1, off  # the bar tells such caches apart
        at += n
    s.close()
    m.close()


@pytest.mark.parametrize("dtype", [Q8_0, Q4_0, F16])
@pytest.mark.parametrize("prec", ["exact", "fast", "fast-f16"])
def test_session_logits(hip_ctx, prec, dtype):
    """A prompt, a second message, a short one of a few tokens, single tokens, and the rest."""
    check(hip_ctx, (40, 35, 7, 1, 1, 26), prec, 4, 2, 64, 3, 110, dtype)


@pytest.mark.parametrize("prec", ["exact", "fast", "fast-f16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(6, 3, 96), (16, 1, 32), (5, 1, 160), (4, 2, 256)])
def test_session_logits_at_head_dims(hip_ctx, heads, kv_heads, hd, prec):
    check(hip_ctx, (45, 9, 1, 1), prec, heads, kv_heads, hd, 2, 56, Q8_0)


@pytest.mark.parametrize("prec,heads,kv_heads,hd", [("fast-f16", 32, 8, 64), ("fast-f16", 32, 4, 128),
                                                    ("fast", 32, 4, 128), ("exact", 32, 4, 128)])
def test_session_logits_of_many_queries(hip_ctx, prec, heads, kv_heads, hd):
    """Chunks that the many-column attention takes (16,384 queries), then a few tokens."""
    check(hip_ctx, (512, 1, 2), prec, heads, kv_heads, hd, 2, 515, Q8_0)


@pytest.mark.parametrize("prec", ["fast-f16", "fast"])
@pytest.mark.parametrize("least,tokens", [(500, 502), (512, 530)])
def test_session_logits_of_a_prompt_on_two_streams(hip_ctx, monkeypatch, least, tokens, prec):
    """From position 13, so that the halves meet inside a tile of the cache: an empty one and 502 tokens (they meet at
    multiples of 256), 256 and 274."""
    monkeypatch.setenv("ALPACA_HIP_SPLIT_MIN", str(least))
    check(hip_ctx, (13, tokens), prec, 32, 8, 64, 2, 13 + tokens, Q8_0)
