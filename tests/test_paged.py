"""What the entry points of the KV cache in pages and of token log probabilities
refuse, and their size arithmetic: checked before any device call, so on the CPU."""
import ctypes as C

import pytest

from alpaca_amd import _lib as L
from alpaca_amd import kvcache, sampling
from alpaca_amd.kvcache import PAGED_WORKSPACE_ZERO, PagedBatch, PagedCache
from tests.test_kv_q4_cache import made  # noqa: F401  (the stand-in for the library's allocator)

# Stands for a context (device 0, null stream) in calls that are refused before they use it.
CTX = C.create_string_buffer(64)
ctx = C.addressof(CTX)
P = 1 << 20  # a pointer that no refused call follows, 16-byte aligned
F32, F16 = L.F32, L.F16


def refused(rc, what, code=L.INVALID_ARGUMENT):
    assert rc == code
    assert what.encode() in L.lib().ahip_last_error(), L.lib().ahip_last_error()


def test_cache_bytes():
    n = C.c_int64()
    for kv_heads, hd, page, pages in ((1, 32, 16, 1), (3, 64, 32, 999), (8, 128, 1024, 1 << 20), (32, 256, 64, 2**31 - 1)):
        assert L.lib().ahip_paged_kv_bytes(kv_heads, hd, page, pages, C.byref(n)) == 0
        assert n.value == kv_heads * hd * page * pages * 2
    for bad in ((0, 64, 16, 1), (1, 48, 16, 1), (1, 288, 16, 1), (1, 64, 8, 1), (1, 64, 24, 1), (1, 64, 2048, 1),
                (1, 64, 0, 1), (1, 64, 16, 0), (1, 64, 16, -1), (40000, 64, 16, 1)):
        assert L.lib().ahip_paged_kv_bytes(*bad, C.byref(n)) == L.INVALID_ARGUMENT
    refused(L.lib().ahip_paged_kv_bytes(32767, 256, 1024, 2**31 - 1, C.byref(n)), "implausibly large")  # past 2^63
    refused(L.lib().ahip_paged_kv_bytes(1, 64, 16, 1, None), "null")


def cache(kc=P, vc=P, kv_heads=2, hd=64, page=16, pages=10):
    return C.byref(L.PagedKVC(kc, vc, kv_heads, hd, page, pages))


def batch(starts=P, lengths=P, table=P, sequences=3, table_stride=8, rows=5, max_rows=0):
    return C.byref(L.PagedBatchC(starts, lengths, table, sequences, table_stride, rows, max_rows))


CACHE = {"kc", "vc", "kv_heads", "hd", "page", "pages"}


def both(kw):
    c = {k: kw.pop(k) for k in list(kw) if k in CACHE}
    return cache(**c), batch(**kw)


def refusals_of_a_batch(call):
    refused(call(ctx=None), "null context")
    refused(call(kc=None), "null cache")
    refused(call(vc=P + 8), "aligned")
    refused(call(hd=80), "head dimension")
    refused(call(page=48), "power of two")
    refused(call(pages=0), "page count")
    refused(call(kv_heads=0), "KV head count")
    refused(call(starts=None), "null batch array")
    refused(call(lengths=None), "null batch array")
    refused(call(table=P + 2), "misaligned batch array")
    refused(call(rows=-1), "batch shape")
    refused(call(rows=2**26 + 1), "batch shape")
    refused(call(sequences=-1), "batch shape")
    refused(call(sequences=2**20 + 1), "batch shape")
    refused(call(max_rows=-1), "batch shape")
    refused(call(table_stride=0), "table's row")
    refused(call(table_stride=2**26 + 1), "table's row")  # past 2^30 positions
    assert call(rows=0, starts=None, lengths=None, table=None) == 0  # nothing to do
    assert call(sequences=0, starts=None, lengths=None, table=None) == 0


def append(ctx=ctx, dtype=F32, q=P, qs=256, qo=P, qos=256, heads=4, k=P, ks=128, v=P, vs=128, rope=P, positions=100,
           **kw):
    c, b = both(kw)
    rows = L.PagedRowsC(q, qo, k, v, qs, qos, ks, vs, rope, positions, 1, dtype, heads)
    return L.lib().ahip_paged_append(ctx, c, b, C.byref(rows), None)


def test_append_refusals():
    refusals_of_a_batch(append)
    refused(L.lib().ahip_paged_append(ctx, cache(), batch(), None, None), "null rows")
    refused(L.lib().ahip_paged_append(ctx, cache(), None, C.byref(L.PagedRowsC()), None), "null batch")
    refused(L.lib().ahip_paged_append(ctx, None, batch(), C.byref(L.PagedRowsC()), None), "null cache")
    for dtype in (L.Q8_0, L.Q4_0, -1, 9):
        refused(append(dtype=dtype), "rows must be")
    refused(append(heads=-1), "query head count")
    refused(append(heads=40000), "query head count")
    refused(append(heads=32767, rows=2**16), "2^30", L.UNSUPPORTED)
    refused(append(rope=P + 4), "rotation table")
    refused(append(positions=0), "rotation table")
    refused(append(k=None), "null keys")
    refused(append(v=P + 2), "values: misaligned")
    refused(append(ks=127), "keys: stride")
    refused(append(vs=1 << 40), "values: implausibly")
    refused(append(q=None), "null queries")
    refused(append(qo=None), "null query output")
    refused(append(heads=0), "queries of no heads")
    refused(append(qos=255), "query output: stride")


def load(ctx=ctx, dtype=F32, k=P, ks=128, v=P, vs=128, **kw):
    c, b = both(kw)
    return L.lib().ahip_paged_load(ctx, c, b, dtype, k, ks, v, vs, None)


def test_load_refusals():
    refusals_of_a_batch(load)
    refused(load(dtype=L.Q4_0), "rows must be")
    refused(load(k=P + 1), "keys: misaligned")
    refused(load(vs=100), "values: stride")
    assert load(k=None, v=None) == 0


def attention(ctx=ctx, dtype=F32, q=P, qs=256, heads=4, window=0, sinks=0, out=P, os=256, ws=P, wb=1 << 40, **kw):
    c, b = both(kw)
    return L.lib().ahip_paged_attention(ctx, c, b, dtype, q, qs, heads, window, sinks, out, os, ws, wb, None)


def test_attention_refusals():
    refusals_of_a_batch(attention)
    refused(attention(dtype=L.Q8_0), "rows must be")
    refused(attention(heads=5), "multiple of the KV heads")
    refused(attention(heads=0), "multiple of the KV heads")
    refused(attention(heads=32766, rows=2**16), "2^30", L.UNSUPPORTED)
    refused(attention(window=-1), "window and sinks")
    refused(attention(window=4, sinks=-1), "window and sinks")
    refused(attention(q=None), "null queries")
    refused(attention(out=None), "null output")
    refused(attention(os=255), "output: stride")
    refused(attention(q=P + 2), "queries: misaligned")
    n = C.c_int64()
    assert L.lib().ahip_paged_attention_workspace(cache(), C.byref(n)) == 0
    refused(attention(ws=None), "workspace, got 0")
    refused(attention(ws=P + 8), "16-byte aligned")
    refused(attention(wb=n.value - 1), f"needs {n.value} bytes")
    refused(L.lib().ahip_paged_attention_workspace(cache(hd=33), C.byref(n)), "head dimension")
    refused(L.lib().ahip_paged_attention_workspace(cache(), None), "null")


def logprobs(ctx=ctx, dtype=F32, logits=P, stride=1000, tokens=P, lp=P, entropy=P, tt=P, tl=P, rows=3, vocab=1000, top=5,
             ws=None, wb=0):
    a = L.LogprobsC(logits, stride, tokens, lp, entropy, tt, tl, dtype, rows, vocab, top)
    return L.lib().ahip_token_logprobs(ctx, C.byref(a), ws, wb, None)


def test_logprobs_refusals():
    refused(logprobs(ctx=None), "null context")
    refused(L.lib().ahip_token_logprobs(ctx, None, None, 0, None), "null arguments")
    refused(logprobs(dtype=L.Q4_0), "rows must be")
    refused(logprobs(rows=-1), "shape")
    refused(logprobs(rows=2**24), "shape")
    refused(logprobs(vocab=0), "shape")
    refused(logprobs(vocab=2**30 + 1, stride=2**30 + 1), "shape")
    refused(logprobs(top=33), "top must be")
    refused(logprobs(top=-1), "top must be")
    refused(logprobs(vocab=4, top=5), "top must be")
    refused(logprobs(logits=None), "null logits")
    refused(logprobs(logits=P + 2), "logits: misaligned")
    refused(logprobs(stride=999), "logits: stride")
    refused(logprobs(tokens=None), "null tokens")
    refused(logprobs(tt=None), "null top outputs")
    refused(logprobs(tl=None), "null top outputs")
    refused(logprobs(lp=P + 2), "misaligned")
    refused(logprobs(tl=P + 2), "misaligned")
    n = C.c_int64()
    assert L.lib().ahip_token_logprobs_workspace(C.byref(n)) == 0
    refused(logprobs(ws=P, wb=n.value - 1), f"{n.value} bytes")
    refused(logprobs(ws=P + 8, wb=n.value), "16-byte aligned")
    refused(L.lib().ahip_token_logprobs_workspace(None), "null")
    assert logprobs(rows=0, logits=None) == 0  # nothing to do
    assert logprobs(lp=None, entropy=None, top=0, logits=None) == 0


def test_the_packed_arguments_are_the_structures_bytes():
    for pack, kind in ((kvcache._PAGED_ROWS, L.PagedRowsC), (sampling._LOGPROBS, L.LogprobsC)):
        values = [P + 64 * i if t is C.c_void_p else 100 + i for i, (_, t) in enumerate(kind._fields_)]
        assert pack(*values) == bytes(kind(*values))


BATCH = PagedBatch(P, P, P, 2, 4, 3)


@pytest.mark.parametrize("fails", [1, 2])
def test_a_cache_that_cannot_be_allocated_keeps_nothing(made, fails):  # noqa: F811
    a, context = made([fails])
    with pytest.raises(L.HIPError) as e:
        PagedCache(context, 10, 2, 64, 16)
    assert e.value.code == L.ALLOC and not a.held


def test_a_workspace_that_cannot_be_allocated_is_allocated_by_the_next_call(made):  # noqa: F811
    a, context = made([3])
    seen = []
    a.ahip_paged_attention = lambda *args: seen.append(args[-3:-1]) or 0
    c = PagedCache(context, 10, 2, 64, 16)
    assert a.held[c._desc.k] == a.held[c._desc.v] == 10 * 2 * 64 * 16 * 2 == c.bytes // 2
    with pytest.raises(L.HIPError):
        c.attention(BATCH, P, P, 4)
    assert not seen and len(a.held) == 2
    c.attention(BATCH, P, P, 4)
    c.attention(BATCH, P, P, 4)
    assert seen == [(c._work, c.workspace_bytes())] * 2 and a.held[c._work] == c.workspace_bytes() > PAGED_WORKSPACE_ZERO
    c.attention(BATCH, P, P, 4, workspace=(P, 5))
    assert seen[-1] == (P, 5)
    c.close()
    c.close()
    assert not a.held


def test_a_closed_context_frees_its_caches_and_their_calls_are_refused(made):  # noqa: F811
    a, context = made()
    a.ahip_paged_attention = lambda *args: 0
    c = PagedCache(context, 10, 2, 64, 16)
    c.attention(BATCH, P, P, 4)
    context.close()
    assert not a.held and a.contexts == 1
    for call in (lambda: c.append(BATCH, P, P), lambda: c.load(BATCH, P, P), lambda: c.workspace_bytes()):
        with pytest.raises(L.InvalidArgument):
            call()


def test_the_log_probabilities_workspace_lives_as_long_as_its_context(made):  # noqa: F811
    a, context = made([1])
    seen = []
    a.ahip_token_logprobs = lambda *args: seen.append(args[2:4]) or 0
    with pytest.raises(L.HIPError):
        sampling.token_logprobs(context, P, 1, 100)
    sampling.token_logprobs(context, P, 1, 100)
    sampling.token_logprobs(context, P, 1, 100)
    assert len(seen) == 2 and seen[0] == seen[1] and list(a.held.items()) == [seen[0]]
    sampling.token_logprobs(context, P, 1, 100, workspace=(P, 9))
    assert seen[-1] == (P, 9)
    context.close()
    assert not a.held
