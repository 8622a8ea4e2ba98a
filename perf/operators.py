"""The operators around a KV cache held in 4 bits, as a serving program calls
them on device tensors, each beside its plain form in elementary torch
operations.

``kind`` "norm_rope": the per-head RMS norm of the queries and keys and their
rotation (``qk_norm_rope``), out of rows that may hold [q | k | v] side by side.

``kind`` "cache": ``tokens`` rows of keys and values written into the cache at
position ``start`` (``Q4Cache.store``) and read back (``Q4Cache.load``).

``kind`` "attend": causal attention of ``tokens`` queries at positions
``start``.. over the cache (``Q4Cache.attention``).

``kind`` "step": one token of a decode loop, its keys and values written and
its queries answered.

The cache holds Q4_0 blocks: 32 values along the head dimension, a scale
d = m / -8 (m the value of largest magnitude, the first of equals) kept as f16,
and n = trunc(x * (1 / d) + 8.5), at most 15; a value reads back as d * (n - 8).
"f32" and "f16" are the type of the rows, queries and outputs.  Head counts and
sizes are those of the benchmark's models (9/3, 15/5 and 32/32 heads of 64) and
generic ones (32/8 heads of 128, odd groups, heads of 32 to 256).
"""
import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
EPS = 1e-5
THETA = 1e5


def _case(kind, dtype, heads, kv_heads, hd, tokens, start=0, **more):
    return dict({"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "hd": hd, "tokens": tokens,
                 "start": start}, **more)


def listed() -> list:
    def named(name, case):
        return dict(case, name=name)
    return [
        # Every layer of a decoded token: launches and latency are all there is.
        named("norm-rope-1", _case("norm_rope", "f32", 9, 3, 64, 1, 2000, interleaved=True)),
        # A message of odd length, read out of the stacked projection's rows.
        named("norm-rope-777", _case("norm_rope", "f32", 15, 5, 64, 777, 1000, interleaved=True)),
        # A long prompt, heads rotated in halves.
        named("norm-rope-4096", _case("norm_rope", "f16", 32, 8, 128, 4096, interleaved=False)),
        # One token's keys and values.
        named("cache-1", _case("cache", "f32", 9, 3, 64, 1, 2000)),
        # A document that starts and ends inside the cache's tiles.
        named("cache-1021", _case("cache", "f32", 15, 5, 64, 1021, 37)),
        # The longest prompt of the benchmark's largest shape.
        named("cache-4096", _case("cache", "f16", 32, 32, 64, 4096)),
        # A decoded token with a short context.
        named("decode-300", _case("attend", "f32", 15, 5, 64, 1, 300)),
        # A decoded token, its keys and values written first, late in a conversation.
        named("step-8000", _case("step", "f32", 9, 3, 64, 1, 8000)),
        # A decoded token far into a long context: the cache's bytes set the time.
        named("decode-131072", _case("attend", "f32", 32, 8, 128, 1, 131071)),
        # A question about a document, in float32.
        named("turn-37-at-1021", _case("attend", "f32", 15, 5, 64, 37, 1021)),
        # A chunk of a prompt through the default batch, the context before it in the cache.
        named("chunk-512-at-3584", _case("attend", "f16", 32, 32, 64, 512, 3584)),
        # A whole prompt at once.
        named("prompt-2048", _case("attend", "f16", 32, 8, 128, 2048)),
    ]


def _log_uniform(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (heads, kv_heads): the benchmark's, and groups of 1 to 16 queries a key
_HEADS = [(9, 3), (15, 5), (32, 32), (32, 8), (16, 1), (12, 12), (14, 2), (24, 8), (40, 8)]
_MOST = 4.0 * 128 * 32 * 2048 * 2049 / 2  # operations of the largest listed attention


def draw(rng) -> dict:
    kind = rng.choice(["norm_rope", "cache", "attend", "attend", "attend", "step"])
    heads, kv_heads = rng.choice(_HEADS)
    hd = rng.choice([64, 64, 64, 128, 128, 128, 32, 96, 160, 256])
    dtype = rng.choice(["f32", "f16"])
    if kind == "norm_rope":
        most = min(8192, 4096 * 40 * 128 // ((heads + kv_heads) * hd))
        return _case(kind, dtype, heads, kv_heads, hd, _log_uniform(rng, 1, most), rng.randint(0, 4000),
                     interleaved=rng.random() < 0.5)
    if kind == "cache":
        most = min(8192, 4096 * 32 * 64 // (kv_heads * hd))
        return _case(kind, dtype, heads, kv_heads, hd, _log_uniform(rng, 1, most), rng.randint(0, 300))
    length = _log_uniform(rng, 1, min(131072, 131072 * 8 * 128 // (kv_heads * hd)))
    tokens = 1
    if kind == "attend" and rng.random() < 0.6:
        tokens = _log_uniform(rng, 2, 2048)
        length = min(max(length, tokens), 32768)
        while 4.0 * hd * heads * tokens * (length - tokens + (tokens + 1) / 2) > _MOST:
            tokens, length = max(1, tokens // 2), max(1, length // 2)
    return _case(kind, dtype, heads, kv_heads, hd, tokens, length - tokens)


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _keys(g, rows, kv_heads, hd, dtype):
    # keys have channels far larger than the rest, in every row
    size = 1 + 5 * (torch.rand(kv_heads, hd, generator=g, device="cuda") < 0.05)
    return (_normal(g, rows, kv_heads, hd) * size).to(TYPES[dtype])


def prepare(case, seed):
    g = _generator(seed)
    H, KVH, hd, T, start, t = (case["heads"], case["kv_heads"], case["hd"], case["tokens"], case["start"],
                               TYPES[case["dtype"]])
    s = {"case": case}
    if case["kind"] == "norm_rope":
        # the stacked projection's rows, [q | k | v] of every token
        rows = _normal(g, T, (H + 2 * KVH) * hd).to(t)
        s["q"], s["k"] = rows[:, :H * hd], rows[:, H * hd:(H + KVH) * hd]
        s["q_gain"], s["k_gain"] = 1 + 0.1 * _normal(g, hd), 1 + 0.1 * _normal(g, hd)
        freq = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        angle = torch.arange(start + T, device="cuda", dtype=torch.float64)[:, None] * freq
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        s["q_out"] = torch.empty(T, H, hd, device="cuda", dtype=t)
        s["k_out"] = torch.empty(T, KVH, hd, device="cuda", dtype=t)
        return s
    if case["kind"] == "cache":
        s["k"], s["v"] = _keys(g, T, KVH, hd, case["dtype"]), _normal(g, T, KVH, hd).to(t)
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return s
    # the rows that the program has written so far, and what the plain form keeps of them
    n = start + T
    s["k"], s["v"] = _keys(g, n, KVH, hd, "f16"), _normal(g, n, KVH, hd).half()
    s["kq"], s["kd"] = _quantise(s["k"])
    s["vq"], s["vd"] = _quantise(s["v"])
    # queries that favour some of the keys, as trained ones do
    s["q"] = (3 * _normal(g, T, H, hd)).to(t)
    s["out"] = torch.empty(T, H, hd, device="cuda", dtype=t)
    if case["kind"] == "step":
        s["k_new"], s["v_new"] = s["k"][start:].to(t), s["v"][start:].to(t)
    return s


# ---------------------------------------------------------------- the plain forms

def _quantise(x):
    """Nibbles (uint8) and scales (f16) of rows [..., hd]."""
    b = x.float().unflatten(-1, (-1, 32))
    m = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = m / -8
    inv = torch.where(d != 0, 1 / d, torch.zeros_like(d))
    return (b * inv + 8.5).floor().clamp(0, 15).to(torch.uint8), d.half()


def _dequantise(n, d):
    return ((n.float() - 8) * d.float()).flatten(-2)


def _norm_rope(x, gain, cs, hd, interleaved):
    x = x.float().unflatten(1, (-1, hd))
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _attend(q, k, v, start):
    """q [T, H, hd], k and v [n, KVH, hd], float32."""
    T, H, hd = q.shape
    n, KVH, _ = k.shape
    G = H // KVH
    rows = q.reshape(T, KVH, G, hd).permute(1, 0, 2, 3).reshape(KVH, T * G, hd)
    s = torch.bmm(rows, k.permute(1, 2, 0).contiguous()) / math.sqrt(hd)
    s = s.view(KVH, T, G, n)
    if T > 1:
        key, pos = torch.arange(n, device="cuda"), start + torch.arange(T, device="cuda")
        s = s.masked_fill_((key[None, :] > pos[:, None])[None, :, None, :], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.bmm(p.view(KVH, T * G, n), v.permute(1, 0, 2).contiguous()).view(KVH, T, G, hd)
    o = o / p.sum(-1, keepdim=True)
    return o.permute(1, 0, 2, 3).reshape(T, H, hd)


# ---------------------------------------------------------------- the framework's calls

@functools.cache
def _context():
    from alpaca_amd.model import HIPContext
    return HIPContext(0)


def _cache(s):
    """The 4-bit cache that the program keeps, holding the rows written so far."""
    if "cache" not in s:
        from alpaca_amd.kvcache import Q4Cache
        c = s["case"]
        s["cache"] = Q4Cache(_context(), c["kv_heads"], c["start"] + c["tokens"], c["hd"])
        if c["kind"] != "cache":
            s["cache"].store(s["k"].data_ptr(), s["v"].data_ptr(), len(s["k"]), 0, "f16")
    return s["cache"]


def _own_run(s):
    c = s["case"]
    T, start, dtype = c["tokens"], c["start"], c["dtype"]
    if c["kind"] == "norm_rope":
        from alpaca_amd.kvcache import qk_norm_rope
        qk_norm_rope(_context(), s["q"].data_ptr(), s["k"].data_ptr(), T, c["heads"], c["kv_heads"], c["hd"],
                     s["q_out"].data_ptr(), s["k_out"].data_ptr(), dtype=dtype, q_gain=s["q_gain"].data_ptr(),
                     k_gain=s["k_gain"].data_ptr(), eps=EPS, rope=s["rope"].data_ptr(), rope_positions=len(s["rope"]),
                     interleaved=c["interleaved"], start=start, q_stride=s["q"].stride(0), k_stride=s["k"].stride(0))
        return [s["q_out"], s["k_out"]]
    cache = _cache(s)
    if c["kind"] == "cache":
        cache.store(s["k"].data_ptr(), s["v"].data_ptr(), T, start, dtype)
        cache.load(s["k_out"].data_ptr(), s["v_out"].data_ptr(), T, start, dtype)
        return [s["k_out"], s["v_out"]]
    if c["kind"] == "step":
        cache.store(s["k_new"].data_ptr(), s["v_new"].data_ptr(), T, start, dtype)
    cache.attention(s["q"].data_ptr(), s["out"].data_ptr(), T, c["heads"], start, dtype)
    return s["out"]


def run(state):
    if own:
        return _own_run(state)
    s, c = state, state["case"]
    t, start = TYPES[c["dtype"]], c["start"]
    if c["kind"] == "norm_rope":
        cs = s["rope"][start:]
        return [_norm_rope(s[x], s[x + "_gain"], cs, c["hd"], c["interleaved"]).to(t) for x in ("q", "k")]
    if c["kind"] == "cache":
        return [_dequantise(*_quantise(s[x])).to(t) for x in ("k", "v")]
    if c["kind"] == "step":
        s["kq"][start:], s["kd"][start:] = _quantise(s["k_new"])
        s["vq"][start:], s["vd"][start:] = _quantise(s["v_new"])
    return _attend(s["q"].float(), _dequantise(s["kq"], s["kd"]), _dequantise(s["vq"], s["vd"]), start).to(t)


# ---------------------------------------------------------------- what a pass has to do

def work(case) -> dict:
    H, KVH, hd, T, start = case["heads"], case["kv_heads"], case["hd"], case["tokens"], case["start"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "norm_rope":
        values = T * (H + KVH) * hd
        # a square and a sum, two scalings, three operations of the rotation for each value
        return {"bytes": 2 * values * size + T * hd * 4 + 2 * hd * 4, "flops": 7 * values}
    if case["kind"] == "cache":
        values = 2 * T * KVH * hd
        # read, written in 4 bits, those read, written
        return {"bytes": values * (2 * size + 2 * 18 / 32), "flops": 6 * values}
    n = start + T
    seen = T * start + T * (T + 1) / 2
    moved = 2 * n * KVH * hd * 18 / 32 + 2 * T * H * hd * size
    if case["kind"] == "step":
        moved += 2 * T * KVH * hd * (size + 18 / 32)
    return {"bytes": moved, "flops": 4 * hd * H * seen}


# ---------------------------------------------------------------- 64-bit results

def _exact_q4(x):
    """What rows [..., hd] read back as: the float32 steps of the format, each exact in 64 bits and then rounded."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    peak = b.abs().max(-1, keepdim=True).values
    first = (b.abs() == peak).int().argmax(-1, keepdim=True)
    d = -b.gather(-1, first) / 8
    safe = torch.where(d == 0, torch.ones_like(d), d)
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / safe).float().double()
    n = ((b * inv).float().double() + 8.5).float().double().trunc().clamp(max=15)
    return (d.half().double() * (n - 8)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    H, KVH, hd, T, start = case["heads"], case["kv_heads"], case["hd"], case["tokens"], case["start"]
    if case["kind"] == "cache":
        return [_exact_q4(s["k"]), _exact_q4(s["v"])]
    if case["kind"] == "norm_rope":
        i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
        turn = (torch.arange(start, start + T, device="cuda", dtype=torch.float64)[:, None] / THETA ** (2 * i / hd))
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]
        out = []
        for name, n in (("q", H), ("k", KVH)):
            x = s[name].double().reshape(T, n, hd)
            x = x / (x.square().sum(-1, keepdim=True) / hd + EPS).sqrt() * s[name + "_gain"].double()
            if case["interleaved"]:
                z = torch.view_as_complex(x.reshape(T, n, hd // 2, 2).contiguous()) * turn
                out.append(torch.view_as_real(z).reshape(T, n, hd))
            else:
                z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
                out.append(torch.cat([z.real, z.imag], -1))
        return out
    k, v = _exact_q4(s["k"]), _exact_q4(s["v"])
    q, out = s["q"].double(), torch.empty(T, H, hd, device="cuda", dtype=torch.float64)
    hidden = torch.ones(T, start + T, device="cuda", dtype=torch.bool).triu(start + 1)
    for h in range(H):
        kv = h // (H // KVH)
        w = (q[:, h] @ k[:, kv].T) * hd ** -0.5
        out[:, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[:, kv]
    return out
