"""The operators of a serving step of many sequences at once, as a serving
program calls them on device tensors, each beside its plain form in elementary
torch operations.

The keys and values of all sequences lie in pages of ``page`` tokens, f16, which
a table gives to every sequence; a step has a number of new tokens of each, side
by side in one batch of rows.

``kind`` "append": the batch's rows [q | k | v] are rotated to their positions,
queries into rows of their own, keys and values into the pages
(``PagedCache.append``); the new positions are read back (``PagedCache.load``).

``kind`` "attend": causal attention of the batch's queries over the pages
(``PagedCache.attention``), of all positions or of the last ``window`` and the
first ``sinks`` ones; pages that no query sees any more have left the table.

``kind`` "step": both, as a layer runs them.

``kind`` "logprobs": of rows of logits the log probabilities of given tokens, the
entropies and the ``top`` likeliest tokens with theirs (``token_logprobs``).

"f32" and "f16" are the type of the rows, queries, outputs and logits.  Head
counts, sizes and the vocabulary are those of the benchmark's models (9/3, 15/5
and 32/32 heads of 64) and generic ones (32/8 heads of 128, odd groups, heads of
32 to 256).
"""
import functools
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16}
THETA = 1e5


def _paged(kind, dtype, heads, kv_heads, hd, page, seqs, longest, chunks=0, tokens=1, window=0, sinks=0,
           interleaved=True, mix=0):
    """``seqs`` sequences of up to ``longest`` tokens, the first ``chunks`` of them with up to ``tokens`` new ones,
    the others with one."""
    return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": page, "seqs": seqs,
            "longest": longest, "chunks": chunks, "tokens": tokens, "window": window, "sinks": sinks,
            "interleaved": interleaved, "mix": mix}


def _logprobs(dtype, rows, vocab, top):
    return {"kind": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top}


def listed() -> list:
    def named(name, case):
        return dict(case, name=name)
    return [
        # One conversation's decoded token, late in it: launches and latency are all there is.
        named("append-1", _paged("append", "f32", 9, 3, 64, 16, 1, 2001)),
        # Three prompts' odd chunks among decoded tokens.
        named("append-48", _paged("append", "f32", 15, 5, 64, 32, 48, 4000, 3, 333)),
        # A long prompt, heads rotated in halves.
        named("append-4096", _paged("append", "f16", 32, 8, 128, 64, 1, 4096, 1, 4096, interleaved=False)),
        # A full batch of decoding conversations of all lengths.
        named("decode-64", _paged("attend", "f16", 32, 8, 128, 16, 64, 8192)),
        # One conversation far into a long context: the pages' bytes set the time.
        named("decode-131072", _paged("attend", "f32", 32, 8, 128, 64, 1, 131072)),
        # Long streams that keep a window and their first tokens.
        named("window-24", _paged("attend", "f32", 15, 5, 64, 32, 24, 60000, window=4096, sinks=4)),
        # A layer's cache and attention of a small model's decoding batch.
        named("step-32", _paged("step", "f32", 9, 3, 64, 16, 32, 2048)),
        # A chunk of a prompt among decoding conversations.
        named("mixed-512", _paged("attend", "f16", 32, 32, 64, 32, 32, 4096, 1, 512)),
        # A whole prompt at once.
        named("prompt-4096", _paged("attend", "f16", 32, 8, 128, 64, 1, 4096, 1, 4096)),
        # Three documents of odd lengths under a window, in float32.
        named("window-2500", _paged("attend", "f32", 24, 8, 128, 128, 3, 6000, 3, 2500, window=1024, sinks=4)),
        # The alternatives that a server shows beside one decoded token.
        named("logprobs-1", _logprobs("f32", 1, 49152, 5)),
        # Scoring a document: every position's logits.
        named("logprobs-2048", _logprobs("f32", 2048, 49152, 20)),
    ]


def _log_uniform(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (heads, kv_heads): the benchmark's, and groups of 1 to 16 queries a key
_HEADS = [(9, 3), (15, 5), (32, 32), (32, 8), (16, 1), (12, 12), (14, 2), (24, 8), (40, 8)]
_MOST = 4.0 * 128 * 32 * 4096 * 4097 / 2  # operations of the largest listed attention


def draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "attend", "attend", "step", "logprobs"])
    dtype = rng.choice(["f32", "f16"])
    if kind == "logprobs":
        vocab = rng.choice([49152, 49152, _log_uniform(rng, 1000, 150000)])
        return _logprobs(dtype, _log_uniform(rng, 1, 2048 * 49152 // max(vocab, 49152)), vocab, rng.randint(0, 20))
    heads, kv_heads = rng.choice(_HEADS)
    hd = rng.choice([64, 64, 64, 128, 128, 128, 32, 96, 160, 256])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    room = 64 * 4096 * 8 * 128 // (kv_heads * hd)  # tokens that all the pages may hold
    seqs = _log_uniform(rng, 1, 128)
    longest = _log_uniform(rng, 1, min(131072, max(1, room // seqs)))
    chunks, tokens, window, sinks = 0, 1, 0, 0
    if rng.random() < 0.5:
        chunks, tokens = rng.randint(1, min(seqs, 4)), _log_uniform(rng, 2, 4096)
    if kind != "append" and rng.random() < 0.4:
        window, sinks = _log_uniform(rng, 1, 8192), rng.choice([0, 0, 1, 4, 40])
    longest = max(longest, tokens)
    while 4.0 * hd * heads * (chunks * tokens + seqs) * min(longest, window + tokens if window else longest) > _MOST / 2:
        tokens, longest, chunks = max(1, tokens // 2), max(1, longest // 2), max(min(chunks, 1), chunks // 2)
    return _paged(kind, dtype, heads, kv_heads, hd, page, seqs, longest, chunks, tokens, window, sinks,
                  rng.random() < 0.5, rng.randint(0, 1 << 30))


def _sequences(case):
    """New tokens and length of every sequence."""
    rng = random.Random(case["mix"])
    new, length = [], []
    for i in range(case["seqs"]):
        new.append((case["tokens"] if i == 0 else rng.randint((case["tokens"] + 1) // 2, case["tokens"]))
                   if i < case["chunks"] else 1)
        least = max(1, case["longest"] // 16)
        length.append(max(new[i], case["longest"] if i == 0 else _log_uniform(rng, least, case["longest"])))
    return new, length


def _first_seen(case, new, length):
    """The first position in the window of any of a sequence's queries."""
    return max(0, length - new - case["window"] + 1) if case["window"] else 0


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _channels(g, kv_heads, hd):
    # keys have channels far larger than the rest, in every row
    return 1 + 5 * (torch.rand(kv_heads, hd, generator=g, device="cuda") < 0.05)


def prepare(case, seed):
    g = _generator(seed)
    t = TYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = _normal(g, rows, vocab).mul_(2.5).to(t)
        s["tokens"] = torch.randint(vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        # every position has some tokens that stand out, the given one often among them
        peaks = torch.randint(vocab, (rows, 4), generator=g, device="cuda")
        peaks[:, 0] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.7, s["tokens"], peaks[:, 0])
        s["logits"].scatter_(1, peaks, (8 + 4 * _normal(g, rows, 4)).to(t))
        s["logprob"] = torch.empty(rows, device="cuda")
        s["entropy"] = torch.empty(rows, device="cuda")
        s["top_tokens"] = torch.empty(rows, top, device="cuda", dtype=torch.int32)
        s["top_logprobs"] = torch.empty(rows, top, device="cuda")
        return s
    H, KVH, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    new, length = _sequences(case)
    S, T = len(new), sum(new)
    # the pages that a sequence holds: all that its queries see, and none between its first tokens and its window
    order = random.Random(seed)
    held = [[p for p in range((n + page - 1) // page)
             if p * page < case["sinks"] or (p + 1) * page > _first_seen(case, m, n) or not case["window"]]
            for m, n in zip(new, length)]
    s["pages"] = sum(map(len, held)) + 3
    ids = list(range(s["pages"]))
    order.shuffle(ids)
    most = max((n + page - 1) // page for n in length)
    table = [[-1] * most for _ in new]
    for row, pages in zip(table, held):
        for p in pages:
            row[p] = ids.pop()
    s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    starts = [sum(new[:i]) for i in range(S + 1)]
    s["row_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(length, dtype=torch.int32, device="cuda")
    # what the plain form takes of a batch: every row's sequence and position
    s["seq"] = torch.repeat_interleave(torch.arange(S), torch.tensor(new)).cuda()
    s["pos"] = torch.cat([torch.arange(n - m, n) for m, n in zip(new, length)]).cuda()
    s["new"], s["rows"], s["max_rows"] = torch.tensor(new).cuda(), T, max(new)
    wide = _channels(g, KVH, hd)
    if case["kind"] != "append":
        # the pages as the steps before have left them
        s["k_pages"] = (_normal(g, s["pages"] * page, KVH, hd) * wide).half()
        s["v_pages"] = _normal(g, s["pages"] * page, KVH, hd).half()
        s["out"] = torch.empty(T, H, hd, device="cuda", dtype=t)
    if case["kind"] == "attend":
        # queries that favour some of the keys, as trained ones do
        s["q"] = (3 * _normal(g, T, H, hd)).to(t)
        return s
    # the stacked projection's rows, [q | k | v] of every token
    rows = _normal(g, T, H + 2 * KVH, hd)
    rows[:, :H] *= 3
    rows[:, H:H + KVH] *= wide
    rows = rows.to(t).view(T, -1)
    s["q"], s["k"], s["v"] = rows[:, :H * hd], rows[:, H * hd:(H + KVH) * hd], rows[:, (H + KVH) * hd:]
    freq = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(max(length), device="cuda", dtype=torch.float64)[:, None] * freq
    s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    s["q_out"] = torch.empty(T, H, hd, device="cuda", dtype=t)
    s["k_out"] = torch.empty(T, KVH, hd, device="cuda", dtype=torch.float16)
    s["v_out"] = torch.empty_like(s["k_out"])
    return s


# ---------------------------------------------------------------- the plain forms

def _rotated(x, cs, hd, interleaved):
    x = x.float().unflatten(1, (-1, hd))
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _attend(s, q, first, last):
    """The rows of sequences first..last-1, padded to the most new tokens and the most visible keys among them."""
    c = s["case"]
    H, KVH, hd, page, S = c["heads"], c["kv_heads"], c["hd"], c["page"], last - first
    new, length = s["new"][first:last], s["lengths"][first:last].long()
    counts, lengths = _sequences(c)
    N = max(counts[first:last])
    seen = [(_first_seen(c, m, n), n) for m, n in zip(counts[first:last], lengths[first:last])]
    V = max(min(c["sinks"], lo) + n - lo for lo, n in seen)
    lo = (length - new - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(length)
    early = lo.clamp(max=c["sinks"])  # sinks ahead of the window
    j = torch.arange(V, device="cuda")[None, :]
    key = torch.where(j < early[:, None], j, j - early[:, None] + lo[:, None])  # [S, V] positions
    inside = key < length[:, None]
    slot = s["table"][first:last].long().gather(1, (key // page).clamp(max=s["table"].shape[1] - 1)) * page + key % page
    slot = torch.where(inside, slot, 0)
    k = s["k_pages"][slot].float().permute(0, 2, 3, 1).reshape(S * KVH, hd, V)  # [.., hd, V]
    v = s["v_pages"][slot].float().permute(0, 2, 1, 3).reshape(S * KVH, V, hd)
    i = torch.arange(N, device="cuda")[None, :]
    row = (s["row_starts"][first:last, None].long() + i).clamp(max=s["rows"] - 1)
    pos = (length - new)[:, None] + i  # [S, N]
    rows = q[row].float().view(S, N, KVH, H // KVH, hd).permute(0, 2, 1, 3, 4).reshape(S * KVH, -1, hd)
    x = torch.bmm(rows, k.contiguous()).div_(math.sqrt(hd)).view(S, KVH, N, H // KVH, V)
    sees = inside[:, None, :] & (key[:, None, :] <= pos[:, :, None])
    if c["window"]:
        sees &= (key[:, None, :] > pos[:, :, None] - c["window"]) | (key[:, None, :] < c["sinks"])
    sees |= (i >= new[:, None])[:, :, None]  # (padding)
    x.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.bmm(p.view(S * KVH, -1, V), v.contiguous()).view(S, KVH, N, H // KVH, hd) / p.sum(-1, keepdim=True)
    return o.permute(0, 2, 1, 3, 4).reshape(S, N, H, hd)[i.expand(S, N) < new[:, None]]


def _attend_all(s, q):
    c = s["case"]
    q = q.view(s["rows"], c["heads"], c["hd"])
    parts = [] if c["chunks"] == 0 else [_attend(s, q, 0, c["chunks"])]
    return torch.cat(parts if c["chunks"] == c["seqs"] else parts + [_attend(s, q, c["chunks"], c["seqs"])])


def _plain_append(s):
    c = s["case"]
    t, cs = TYPES[c["dtype"]], s["rope"][s["pos"]]
    q = _rotated(s["q"], cs, c["hd"], c["interleaved"]).to(t)
    k = _rotated(s["k"], cs, c["hd"], c["interleaved"]).half()
    return q, k, s["v"].float().unflatten(1, (-1, c["hd"])).half()


def _plain_logprobs(s):
    x, top = s["logits"].float() + 0, s["case"]["top"]  # (-0 as 0)
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = (log_total - (e * d).sum(-1, keepdim=True) / total)[:, 0]
    logprob = d.gather(1, s["tokens"][:, None].long()) - log_total
    # whole numbers in the order of the logits, a lower index ahead of a higher one of the same value
    u = x.view(torch.int32)
    u = torch.where(u < 0, u ^ 0x7FFFFFFF, u).long()
    key = u * (1 << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device="cuda"))
    best = x.shape[1] - 1 - key.topk(top, -1).values % (1 << 32)
    return [logprob[:, 0], entropy, best.int(), d.gather(1, best) - log_total]


# ---------------------------------------------------------------- the framework's calls

@functools.cache
def _context():
    from alpaca_amd.model import HIPContext
    return HIPContext(0)


def _cache(s):
    """The pages that the program keeps, holding what was written so far, and the step's batch."""
    if "cache" not in s:
        from alpaca_amd.kvcache import PagedBatch, PagedCache
        c = s["case"]
        s["cache"] = PagedCache(_context(), s["pages"], c["kv_heads"], c["hd"], c["page"])
        if c["kind"] != "append":
            # all pages in order, as one long sequence
            n = s["pages"] * c["page"]
            every = torch.arange(s["pages"], dtype=torch.int32, device="cuda")
            ends = torch.tensor([0, n, n], dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()  # (the context has a stream of its own)
            fill = PagedBatch(ends.data_ptr(), ends[1:].data_ptr(), every.data_ptr(), 1, s["pages"], n, n)
            s["cache"].append(fill, s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), dtype="f16")
            torch.cuda.synchronize()
        s["batch"] = PagedBatch(s["row_starts"].data_ptr(), s["lengths"].data_ptr(), s["table"].data_ptr(), c["seqs"],
                                s["table"].shape[1], s["rows"], s["max_rows"])
    return s["cache"]


def _own_run(s):
    c = s["case"]
    if c["kind"] == "logprobs":
        from alpaca_amd.sampling import token_logprobs
        token_logprobs(_context(), s["logits"].data_ptr(), c["rows"], c["vocab"], tokens=s["tokens"].data_ptr(),
                       logprobs=s["logprob"].data_ptr(), entropy=s["entropy"].data_ptr(), top=c["top"],
                       top_tokens=s["top_tokens"].data_ptr(), top_logprobs=s["top_logprobs"].data_ptr(),
                       dtype=c["dtype"])
        return [s["logprob"], s["entropy"], s["top_tokens"], s["top_logprobs"]]
    cache = _cache(s)
    batch = s["batch"]
    if c["kind"] == "attend":
        cache.attention(batch, s["q"].data_ptr(), s["out"].data_ptr(), c["heads"], c["dtype"], window=c["window"],
                        sinks=c["sinks"])
        return s["out"]
    stride = s["q"].stride(0)
    cache.append(batch, s["k"].data_ptr(), s["v"].data_ptr(), s["q"].data_ptr(), s["q_out"].data_ptr(), c["heads"],
                 c["dtype"], rope=s["rope"].data_ptr(), rope_positions=len(s["rope"]), interleaved=c["interleaved"],
                 q_stride=stride, k_stride=stride, v_stride=stride)
    if c["kind"] == "append":
        cache.load(batch, s["k_out"].data_ptr(), s["v_out"].data_ptr(), "f16")
        return [s["q_out"], s["k_out"], s["v_out"]]
    cache.attention(batch, s["q_out"].data_ptr(), s["out"].data_ptr(), c["heads"], c["dtype"], window=c["window"],
                    sinks=c["sinks"])
    return [s["q_out"], s["out"]]


def run(state):
    if own:
        return _own_run(state)
    s, c = state, state["case"]
    if c["kind"] == "logprobs":
        return _plain_logprobs(s)
    if c["kind"] == "attend":
        return _attend_all(s, s["q"]).to(TYPES[c["dtype"]])
    q, k, v = _plain_append(s)
    if c["kind"] == "append":
        return [q, k, v]
    slot = s["table"][s["seq"], s["pos"] // c["page"]].long() * c["page"] + s["pos"] % c["page"]
    s["k_pages"][slot], s["v_pages"][slot] = k, v
    return [q, _attend_all(s, q).to(TYPES[c["dtype"]])]


# ---------------------------------------------------------------- what a pass has to do

def work(case) -> dict:
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # a maximum, a difference, an exponential, two sums and a product for each logit
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    H, KVH, hd = case["heads"], case["kv_heads"], case["hd"]
    new, length = _sequences(case)
    T = sum(new)
    moved = flops = 0
    if case["kind"] != "attend":
        # [q | k | v] read, q written, k and v written as f16, the table's rows
        moved += T * (2 * H + 2 * KVH) * hd * size + T * 2 * KVH * hd * 2 + T * hd * 4
        flops += 3 * T * (H + KVH) * hd
    if case["kind"] == "append":
        return {"bytes": moved + 2 * T * 2 * KVH * hd * 2, "flops": flops}  # read and written once more
    for m, n in zip(new, length):
        lo = _first_seen(case, m, n)
        moved += 2 * 2 * KVH * hd * (n - lo + min(case["sinks"], lo)) + 2 * m * H * hd * size
        for i in range(n - m, n):  # (the query's keys)
            a = max(0, i - case["window"] + 1) if case["window"] else 0
            flops += 4 * hd * H * (i + 1 - a + min(case["sinks"], a))
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------- 64-bit results

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        logprob, entropy, tokens, tops = [], [], [], []
        for x, y in zip(s["logits"].split(256), s["tokens"].split(256)):
            lp = torch.log_softmax(x.double(), -1)
            logprob.append(lp.gather(1, y.long()[:, None])[:, 0])
            entropy.append(-(lp.exp() * lp).sum(-1))
            best = x.double().sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            tokens.append(best.int())
            tops.append(lp.gather(1, best))
        return [torch.cat(z) for z in (logprob, entropy, tokens, tops)]
    H, KVH, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    new, length = _sequences(case)
    q = s["q"].double().reshape(-1, H, hd)
    head = []
    if case["kind"] != "attend":
        i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
        turn = s["pos"].double()[:, None] / THETA ** (2 * i / hd)
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]

        def rotated(x):
            if case["interleaved"]:
                z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn
                return torch.view_as_real(z).flatten(-2)
            z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)
        q, k = rotated(q), rotated(s["k"].double().reshape(-1, KVH, hd))
        v = s["v"].double().reshape(-1, KVH, hd)
        if case["kind"] == "append":
            return [q, k, v]
        head = [q]
        q = q.to(TYPES[case["dtype"]]).double()  # as the rows of the second operator hold them
    # the pages are held in f16 by definition
    kp, vp = s["k_pages"].view(-1, page, KVH, hd), s["v_pages"].view(-1, page, KVH, hd)
    table, out, at = s["table"].long(), [], 0
    for r, (m, n) in enumerate(zip(new, length)):
        lo = _first_seen(case, m, n) // page
        pages = [p for p in range((n + page - 1) // page) if p * page < case["sinks"] or p >= lo]
        where = torch.cat([torch.arange(p * page, (p + 1) * page) for p in pages]).cuda()
        ids = table[r, torch.tensor(pages).cuda()]
        ks, vs = kp[ids].flatten(0, 1).double(), vp[ids].flatten(0, 1).double()
        mine = torch.arange(n - m, n, device="cuda")
        if case["kind"] == "step":
            new_at = torch.searchsorted(where, mine)
            ks[new_at], vs[new_at] = k[at:at + m].half().double(), v[at:at + m].half().double()
        hidden = where[None, :] > mine[:, None]
        if case["window"]:
            hidden |= (where[None, :] <= mine[:, None] - case["window"]) & (where[None, :] >= case["sinks"])
        o = torch.empty(m, H, hd, device="cuda", dtype=torch.float64)
        for h in range(H):
            w = (q[at:at + m, h] @ ks[:, h // (H // KVH)].T.contiguous()) * hd ** -0.5
            o[:, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ vs[:, h // (H // KVH)].contiguous()
        out.append(o)
        at += m
    return head + [torch.cat(out)] if head else torch.cat(out)
