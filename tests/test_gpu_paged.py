"""The KV cache in pages on the GPU: writing with the rotation and reading back,
and the attention of ragged batches over it, against 64-bit plain forms."""
import ctypes as C

import numpy as np
import pytest

from alpaca_amd import _lib as L
from alpaca_amd.kvcache import PAGED_WORKSPACE_ZERO, PagedBatch, PagedCache, rope_table
from tests import paged_reference as ref
from tests.paged_reference import NP, Batch
from tests.q4_reference import Device

pytestmark = pytest.mark.gpu


def rows(rng, tokens, heads, hd, dtype, size=1.0):
    return (rng.standard_normal((tokens, heads, hd)) * size).astype(NP[dtype])


def padded(x, extra, lead=0, fill=7.0):
    """Rows with `extra` elements behind each one's and `lead` ahead of the first, flat, and their stride."""
    flat = x.reshape(len(x), -1)
    w = flat.shape[1] + extra
    out = np.full(lead + len(x) * w, fill, x.dtype)
    out[lead:].reshape(len(x), w)[:, :flat.shape[1]] = flat
    return out, w


def garbage(ctx, cache):
    """Makes all that was never written NaN."""
    for p in (cache._desc.k, cache._desc.v):
        L.check(L.lib().ahip_memset(ctx.handle, p, 0xFF, cache.bytes // 2))


def make(hip_ctx, batch, kv_heads, hd):
    c = PagedCache(hip_ctx, batch.pages, kv_heads, hd, batch.page)
    garbage(hip_ctx, c)
    return c


class Rows:
    """Rows of a type on the device, `extra` elements apart and `lead` from where they could lie; what lies between them
    stays."""

    def __init__(self, dev, count, width, dtype, extra=0, lead=0):
        self.dev, self.count, self.width, self.dtype, self.extra, self.lead = dev, count, width, dtype, extra, lead
        self.stride, self.size = width + extra, NP[dtype]().nbytes
        self.base = dev.empty((lead + count * self.stride) * self.size)
        self.p = self.base + lead * self.size

    def get(self, heads):
        a = self.dev.get(self.base, self.lead + self.count * self.stride, NP[self.dtype])
        assert (a[:self.lead].view(np.uint8) == 0xA5).all()
        a = a[self.lead:].reshape(self.count, self.stride)
        assert (np.ascontiguousarray(a[:, self.width:]).view(np.uint8) == 0xA5).all()
        return a[:, :self.width].reshape(self.count, heads, -1)


def untouched(x):
    return (np.ascontiguousarray(x).view(np.uint8) == 0xA5).all()


def append(dev, cache, on, k, v, dtype, extra=0, lead=0, **kw):
    size = NP[dtype]().nbytes
    (kp, ks), (vp, vs) = padded(k, extra, lead), padded(v, extra, lead)
    cache.append(on, dev.put(kp) + lead * size, dev.put(vp) + lead * size, dtype=dtype, k_stride=ks, v_stride=vs, **kw)


def load(dev, cache, on, count, dtype, extra=0, lead=0):
    w = cache.kv_heads * cache.head_dim
    out = [Rows(dev, count, w, dtype, extra, lead) for _ in range(2)]
    cache.load(on, out[0].p, out[1].p, dtype, k_stride=w + extra, v_stride=w + extra)
    return [r.get(cache.kv_heads) for r in out]


def as_held(x):
    with np.errstate(over="ignore"):
        return x.astype(np.float16)


# ---------------------------------------------------------------- append, load

SHAPES = [  # new, lengths
    ([1], [1]), ([16], [16]), ([17], [33]), ([1, 1, 1], [15, 16, 17]), ([5, 0, 40, 1], [5, 20, 77, 130]),
    ([0, 0, 3], [0, 9, 3]), ([7, 8, 9, 200], [31, 32, 33, 257])]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page,kv_heads,heads", [(32, 16, 1, 3), (64, 32, 3, 9), (96, 16, 5, 5), (128, 64, 8, 32),
                                                    (160, 128, 2, 2), (192, 16, 1, 16), (224, 256, 3, 3), (256, 1024, 2, 4)])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_append_rotates_and_load_reads_back(hip_ctx, case, hd, page, kv_heads, heads, dtype):
    check_append(hip_ctx, case, *SHAPES[case], hd, page, kv_heads, heads, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page,kv_heads,heads,new,lengths", [
    (64, 32, 32, 32, [1100], [1500]), (128, 16, 8, 40, [700, 0, 333, 90], [700, 5, 1000, 99]), (160, 64, 3, 7, [2100], [2101]),
    (256, 16, 1, 9, [1030], [1030]), (128, 16, 8, 33, [1] * 520, [1 + i % 70 for i in range(520)])])
def test_append_of_many_tokens(hip_ctx, hd, page, kv_heads, heads, new, lengths, dtype):
    for case in range(3):
        check_append(hip_ctx, case, new, lengths, hd, page, kv_heads, heads, dtype)


def check_append(hip_ctx, case, new, lengths, hd, page, kv_heads, heads, dtype):
    rng = np.random.default_rng(100 * hd + case)
    b = Batch(rng, page, new, lengths, spare_rows=case % 3, lead=case % 2)
    extra, lead = [(0, 0), (16, 0), (3, 1)][case % 3]  # rows on 16 bytes, apart, and at any element
    q, k, v = (rows(rng, b.rows, n, hd, dtype, 3) for n in (heads, kv_heads, kv_heads))
    table, interleaved = rope_table(max(lengths), hd, 1e4), case % 2 == 0
    cache = make(hip_ctx, b, kv_heads, hd)
    with Device(hip_ctx) as dev:
        on = b.on(dev)
        qp, qs = padded(q, extra, lead)
        out = Rows(dev, b.rows, heads * hd, dtype, extra, lead)
        append(dev, cache, on, k, v, dtype, extra, lead, q=dev.put(qp) + lead * q.itemsize, q_out=out.p, heads=heads,
               rope=dev.put(table), rope_positions=len(table), interleaved=interleaved, q_stride=qs, q_out_stride=qs)
        got_q = out.get(heads)
        got32, got16 = load(dev, cache, on, b.rows, "f32", extra, lead), load(dev, cache, on, b.rows, "f16", extra, lead)
    cache.close()
    for a in (got_q, *got32, *got16):  # rows of no sequence
        assert untouched(a[:b.lead]) and untouched(a[b.starts[-1]:])
    mine = slice(b.lead, b.starts[-1])
    if b.starts[-1] == b.lead:
        return
    pos = np.array([p for _, p in b.positions()])
    assert np.array_equal(got16[0][mine].astype(np.float32), got32[0][mine])
    assert np.array_equal(got16[1][mine].astype(np.float32), got32[1][mine])
    assert np.array_equal(got16[1][mine], as_held(v[mine]))
    want, off = ref.rotated(k[mine], pos, table, interleaved)
    assert (np.abs(got32[0][mine] - want) <= off + ref.half_step(np.abs(want) + off, "f16")).all()
    want, off = ref.rotated(q[mine], pos, table, interleaved)
    assert (np.abs(got_q[mine].astype(np.float64) - want) <= off + ref.half_step(np.abs(want) + off, dtype)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_append_without_rotation_or_queries_keeps_values(hip_ctx, dtype):
    rng = np.random.default_rng(1)
    b = Batch(rng, 16, [40, 3], [50, 90])
    q, k, v = (rows(rng, b.rows, n, 64, dtype) for n in (4, 2, 2))
    cache = make(hip_ctx, b, 2, 64)
    with Device(hip_ctx) as dev:
        on = b.on(dev)
        append(dev, cache, on, k, v, dtype)
        assert all(np.array_equal(g, as_held(x)) for g, x in zip(load(dev, cache, on, b.rows, "f16"), (k, v)))
        place = dev.put(q)  # queries without a table: copied, in place: as they were
        append(dev, cache, on, k, v, dtype, q=place, q_out=place, heads=4)
        assert np.array_equal(dev.get(place, q.shape, q.dtype), q)
        table = rope_table(90, 64, 1e4)
        out = Rows(dev, b.rows, 4 * 64, dtype)
        kw = dict(heads=4, rope=dev.put(table), rope_positions=90)
        append(dev, cache, on, k, v, dtype, q=place, q_out=out.p, **kw)
        append(dev, cache, on, k, v, dtype, q=place, q_out=place, **kw)
        assert np.array_equal(dev.get(place, q.shape, q.dtype), out.get(4))
    cache.close()


def test_positions_that_are_not_written_keep_their_bytes(hip_ctx):
    rng = np.random.default_rng(2)
    b = Batch(rng, 32, [100, 70, 5], [100, 70, 5])
    held = {}
    cache = make(hip_ctx, b, 3, 96)
    with Device(hip_ctx) as dev:
        k, v = (rows(rng, b.rows, 3, 96, "f16") for _ in range(2))
        append(dev, cache, b.on(dev), k, v, "f16")
        for i, sp in enumerate(b.positions()):
            held[sp] = k[i], v[i]
        for new, lengths in (([1, 1, 1], [38, 64, 5]), ([20, 0, 2], [70, 0, 3]), ([32, 16, 0], [64, 48, 5])):
            s = Batch(rng, 32, new, lengths, b.pages, stride=b.stride)
            s.table = b.table
            k, v = (rows(rng, s.rows, 3, 96, "f16") for _ in range(2))
            append(dev, cache, s.on(dev), k, v, "f16")
            for i, sp in enumerate(s.positions()):
                held[sp] = k[i], v[i]
            got = load(dev, cache, b.on(dev), b.rows, "f16")
            for g, want in zip(got, zip(*(held[sp] for sp in b.positions()))):
                assert np.array_equal(g, np.stack(want))
        # what lies behind the sequences in their pages, and the other pages
        ends = [-(-n // 32) * 32 for n in b.lengths]
        rest = Batch(rng, 32, [e - n for e, n in zip(ends, b.lengths)], ends, b.pages, stride=b.stride)
        rest.table = b.table
        assert rest.rows and all(np.isnan(x).all() for x in load(dev, cache, rest.on(dev), rest.rows, "f32"))
        unused = [i for i in range(b.pages) if i not in b.table]
        for p in (cache._desc.k, cache._desc.v):
            assert (dev.get(p, cache.bytes // 2, np.uint8).reshape(b.pages, -1)[unused] == 0xFF).all()
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 70000.0])
def test_a_token_without_a_form_is_nan_in_its_head_only(hip_ctx, dtype, value):
    rng = np.random.default_rng(3)
    b = Batch(rng, 16, [40], [45])
    k, v = rows(rng, 40, 2, 64, dtype), rows(rng, 40, 2, 64, dtype)
    with np.errstate(over="ignore"):
        k[7, 1, 63], v[20, 0, 0] = value, value
    cache = make(hip_ctx, b, 2, 64)
    with Device(hip_ctx) as dev:
        on = b.on(dev)
        append(dev, cache, on, k, v, dtype)
        got = load(dev, cache, on, 40, "f32")
    cache.close()
    odd = np.zeros((40, 2), bool)
    odd[7, 1] = odd[20, 0] = True
    for g, x in zip(got, (k, v)):
        assert np.isnan(g[odd]).all() and np.array_equal(g[~odd], as_held(x)[~odd].astype(np.float32))


def test_positions_without_a_place_store_nothing(hip_ctx):
    """Past the rotation's table, past the pages' table, in pages that there are not, below 0."""
    rng = np.random.default_rng(4)
    b = Batch(rng, 16, [40, 30, 20], [60, 30, 12], stride=3)
    b.table[1, 1], b.table[1, 0] = -7, b.pages
    k, v, q = rows(rng, b.rows, 2, 64, "f32"), rows(rng, b.rows, 2, 64, "f32"), rows(rng, b.rows, 4, 64, "f32")
    cache = make(hip_ctx, b, 2, 64)
    with Device(hip_ctx) as dev:
        on = b.on(dev)
        out = Rows(dev, b.rows, 256, "f32")
        append(dev, cache, on, k, v, "f32", q=dev.put(q), q_out=out.p, heads=4, rope=dev.put(rope_table(44, 64, 1e4)),
               rope_positions=44)
        got_k, got_v = load(dev, cache, on, b.rows, "f32")
        got_q = out.get(4)
    cache.close()
    for i, (s, p) in enumerate(b.positions()):
        turned = 0 <= p < 44
        assert np.isnan(got_q[i]).all() == (not turned) and np.isfinite(got_q[i]).all() == turned
        place = turned and (s != 1 or p >= 32) and p < 48
        assert np.isfinite(got_k[i]).all() == place and np.isnan(got_k[i]).all() == (not place), (s, p)
        assert np.isfinite(got_v[i]).all() == place and np.isnan(got_v[i]).all() == (not place), (s, p)


# ---------------------------------------------------------------- attention

def fill(dev, cache, rng, batch, k_size=1.0, v_size=1.0):
    """Every position of the batch's sequences, with some channels of the keys far larger; the values by sequence."""
    w = ref.whole(rng, batch)
    k, v = (rows(rng, w.rows, cache.kv_heads, cache.head_dim, "f16", n) for n in (k_size, v_size))
    k *= (1 + 5 * (rng.random((cache.kv_heads, cache.head_dim)) < 0.05)).astype(np.float16)
    if w.rows:
        append(dev, cache, w.on(dev), k, v, "f16")
    return [(k[w.sequence_rows(s)], v[w.sequence_rows(s)]) for s in range(len(w.new))]


def attend(dev, cache, on, q, dtype, extra=0, lead=0, **kw):
    T, H, hd = q.shape
    qp, qs = padded(q, extra, lead)
    out = Rows(dev, T, H * hd, dtype, extra, lead)
    cache.attention(on, dev.put(qp) + lead * q.itemsize, out.p, H, dtype, q_stride=qs, out_stride=qs, **kw)
    return out.get(H)


def check(got, q, data, batch, dtype, label, window=0, sinks=0, heads=None):
    worst = 0.0
    assert untouched(got[:batch.lead]) and untouched(got[batch.starts[-1]:])
    for s, (m, n) in enumerate(zip(batch.new, batch.lengths)):
        r = batch.sequence_rows(s)
        want, bound = ref.attention(q[r], *data[s], n - m, dtype, window, sinks, heads)
        pick = slice(None) if heads is None else heads
        off = np.abs(got[r][:, pick].astype(np.float64) - want[:, pick])
        near = bool((off <= bound[:, pick]).all())  # (a NaN is not)
        if m:
            worst = max(worst, np.max(off / np.maximum(bound[:, pick], 1e-300)) if near else np.inf)
        assert near, (label, s, m, n, np.nanmax(off), np.isnan(off).sum())
    print(f"[attention] {label}: {worst:.3f} of the bound")


def attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, extra=0, lead=0, window=0, sinks=0, hint=True,
                   seed=0, q_size=3.0, some_heads=None, spare_rows=2):
    rng = np.random.default_rng(heads * 7919 + hd * 31 + sum(lengths) + seed)

    def held(s, p):  # a sequence's pages: those that its queries see
        lo = max(0, lengths[s] - new[s] - window + 1) if window else 0
        return p * page < sinks or (p + 1) * page > lo or not window
    b = Batch(rng, page, new, lengths, spare_rows=spare_rows)
    q = rows(rng, b.rows, heads, hd, dtype, q_size)
    cache = make(hip_ctx, b, kv_heads, hd)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        if window:  # the others' are given away, and hold NaN
            for s in range(len(new)):
                for p in range(b.stride):
                    if p * page < lengths[s] and not held(s, p):
                        i = b.table[s, p]
                        for buf in (cache._desc.k, cache._desc.v):
                            n = cache.bytes // 2 // b.pages
                            L.check(L.lib().ahip_memset(hip_ctx.handle, buf + int(i) * n, 0xFF, n))
                        b.table[s, p] = [-1, i, 2**31 - 1][(s + p) % 3]
        got = attend(dev, cache, b.on(dev, hint), q, dtype, extra, lead, window=window, sinks=sinks)
        if cache._work:
            assert not dev.get(cache._work, PAGED_WORKSPACE_ZERO, np.uint8).any()
    cache.close()
    check(got, q, data, b, dtype, (heads, kv_heads, hd, page, new, lengths, dtype, window, sinks), window, sinks, some_heads)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 32, 256])
def test_attention_at_every_head_dim(hip_ctx, hd, page, dtype):
    attention_case(hip_ctx, 6, 2, hd, page, [1, 5, 37, 1], [101, 35, 102, 1], dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (4, 4), (16, 1), (17, 1), (14, 2), (40, 1), (40, 8)])
@pytest.mark.parametrize("new,lengths", [([1, 1], [32, 701]), ([3, 0, 18], [3, 50, 51])])
def test_attention_at_groups_of_query_heads(hip_ctx, heads, kv_heads, new, lengths, dtype):
    attention_case(hip_ctx, heads, kv_heads, 64, 32, new, lengths, dtype, extra=8)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_around_tile_and_page_edges(hip_ctx, page, dtype):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1023, 1024, 1025]
    attention_case(hip_ctx, 4, 2, 128, page, [1] * len(lengths), lengths, dtype)
    attention_case(hip_ctx, 4, 2, 128, page, [min(n, 1 + i % 16) for i, n in enumerate(lengths)], lengths, dtype, extra=3,
                   lead=1)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,hd,page,new,lengths", [
    (9, 3, 64, 16, [1], [8001]), (32, 8, 128, 64, [1], [4096]), (2, 1, 64, 1024, [1], [40001]),
    (9, 3, 64, 32, [11, 1, 1], [3011, 9000, 77]), (4, 1, 96, 16, [40], [5040]), (8, 1, 256, 16, [1, 1], [30000, 12])])
def test_attention_over_long_sequences(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype):
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_many_sequences(hip_ctx, dtype):
    """More than a wave's lanes, some without rows."""
    rng = np.random.default_rng(5)
    lengths = [int(n) for n in rng.integers(1, 400, 150)]
    new = [int(min(n, rng.integers(0, 4))) for n in lengths]
    attention_case(hip_ctx, 4, 2, 64, 16, new, lengths, dtype)
    attention_case(hip_ctx, 4, 2, 64, 16, new, lengths, dtype, hint=False, window=50, sinks=3)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("sequences,kv_heads,longest", [(2, 2, 20000), (20, 1, 8000), (64, 1, 3000), (65, 1, 3000), (100, 1, 2500),
                                                        (140, 1, 2000)])
def test_attention_split_evenly_whatever_the_lengths(hip_ctx, sequences, kv_heads, longest, dtype):
    """Shares of more than a few steps, below and above a wave's lanes and half of the workgroups."""
    rng = np.random.default_rng(sequences)
    lengths = [longest] + [int(n) for n in rng.integers(longest // 3, longest, sequences - 1)]
    attention_case(hip_ctx, 2 * kv_heads, kv_heads, 64, 32, [1] * sequences, lengths, dtype)


# (heads, kv_heads, hd, page, new, lengths): chips full of workgroups of 128 and 64 columns, with sequences of few
# columns among them (tests/paged_shapes.py has shapes for every kernel, those of 256 columns too)
WIDE = [(64, 64, 64, 16, [700, 1, 513], [700, 300, 600]), (96, 96, 32, 64, [300, 5, 410], [431, 6, 410]),
        (80, 80, 96, 32, [1, 900], [700, 901]), (64, 32, 128, 16, [550, 1, 2], [1100, 33, 64]),
        (64, 32, 128, 1024, [1100], [1100]), (32, 32, 64, 32, [512, 1, 1], [900, 44, 1000]),
        (32, 8, 128, 64, [260, 30], [300, 31]), (24, 8, 64, 16, [170, 1], [1800, 5])]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_attention_of_many_columns(hip_ctx, case, dtype):
    heads, kv_heads, hd, page, new, lengths = WIDE[case]
    some = [0, heads // 2, heads - 1]
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, extra=[0, 8, 3][case % 3], lead=case % 2,
                   some_heads=some)
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, hint=False, window=100, sinks=[0, 5, 70][case % 3],
                   some_heads=some)


# turns of a long context, whose keys workgroups share, with shorter sequences among them
TURNS = [(32, 8, 128, 64, [200], [4200]), (32, 8, 128, 16, [150, 1, 1], [3000, 2100, 7]), (16, 4, 96, 32, [400], [2500]),
         (24, 8, 96, 16, [180, 17], [2048, 1700]), (32, 8, 128, 128, [100] + [1] * 31, [4000] + [9] * 31),
         (64, 8, 128, 16, [90], [90]), (16, 16, 128, 16, [70, 70, 70], [70, 1100, 2200])]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 4), (20, 0)])
@pytest.mark.parametrize("case", range(len(TURNS)))
def test_attention_of_turns_of_a_long_context(hip_ctx, case, window, sinks, dtype):
    heads, kv_heads, hd, page, new, lengths = TURNS[case]
    some = [0, heads // 2, heads - 1]
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, extra=[0, 8, 3][case % 3], lead=case % 2,
                   window=window, sinks=sinks, some_heads=some)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [160, 192, 224, 256])
def test_attention_of_many_columns_of_wide_heads(hip_ctx, hd, dtype):
    attention_case(hip_ctx, 64, 64, hd, 32, [600, 1], [650, 3], dtype, some_heads=[0, 33])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 16), (100, 40), (4096, 4), (2**31 - 1, 0),
                                          (64, 2**31 - 1)])
def test_windows(hip_ctx, window, sinks, page, dtype):
    attention_case(hip_ctx, 6, 2, 64, page, [1, 1, 20, 3, 0, 1], [1, 500, 300, 3, 40, 200], dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-6, 1, 1), (60, 4, 1), (1, 1, 1e-4), (1, 1e-4, 3000), (1, 300, 1),
                                                  (0, 1, 1)])
@pytest.mark.parametrize("new", [3, 300])
def test_attention_of_small_and_large_values(hip_ctx, q_size, k_size, v_size, new, dtype):
    """Near-uniform and one-hot softmaxes, values near both ends of f16; with few columns and with many."""
    rng = np.random.default_rng(11)
    H = 6 if new == 3 else 64
    b = Batch(rng, 32, [new], [new + 200])
    q = rows(rng, new, H, 64, dtype, q_size)
    cache = make(hip_ctx, b, H // 2, 64)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b, k_size, v_size)
        got = attend(dev, cache, b.on(dev), q, dtype)
    cache.close()
    check(got, q, data, b, dtype, (q_size, k_size, v_size, new, dtype), heads=[0, H - 1])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new", [2, 300])
def test_scores_past_the_exponent_s_precision(hip_ctx, new, dtype):
    """Keys and queries of 1e4: scores of 1e9 or more.  Of a row whose keys are one key times 1, 0.5 and 0.25, all but
    the largest have no weight, so the output is the mean of those values, exactly as many as there are."""
    rng = np.random.default_rng(12)
    H, hd = (4, 64) if new == 2 else (64, 64)
    n = new + 100
    b = Batch(rng, 16, [new], [n])
    base = (rng.choice([-1.0, 1.0], hd) * 8192).astype(np.float16)
    scale = np.array([1.0, 0.5, 0.25])[rng.integers(0, 3, n)]
    scale[0] = 1.0
    k = np.broadcast_to((base * scale[:, None]).astype(np.float16)[:, None], (n, H, hd)).copy()
    v = rows(rng, n, H, hd, "f16")
    q = np.broadcast_to(base.astype(NP[dtype]), (new, H, hd)).copy()
    cache = make(hip_ctx, b, H, hd)
    with Device(hip_ctx) as dev:
        append(dev, cache, ref.whole(rng, b).on(dev), k, v, "f16")
        got = attend(dev, cache, b.on(dev), q, dtype)
    cache.close()
    for t in range(new):
        top = [j for j in range(n - new + t + 1) if scale[j] == 1]
        want = v[top, :].astype(np.float64).mean(0)
        # equal weights: what the sums and the output's rounding lose
        off = (len(top) + 8) * 2.0 ** -24 * np.abs(v[top].astype(np.float64)).mean(0) + ref.half_step(want, dtype)
        assert (np.abs(got[t] - want) <= off * 1.01).all(), t


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("heads,tokens", [(4, 1), (4, 5), (64, 300)])
def test_a_token_without_a_form_reaches_only_the_queries_that_see_it(hip_ctx, where, heads, tokens, dtype):
    rng = np.random.default_rng(13)
    start, n = 60, 60 + tokens
    KVH = heads // 2
    b = Batch(rng, 16, [tokens], [n])
    k, v = rows(rng, n, KVH, 64, "f16"), rows(rng, n, KVH, 64, "f16")
    q = rows(rng, tokens, heads, 64, dtype)
    hit = start + tokens // 2
    clean = k.copy(), v.copy()
    (k if where == "k" else v)[hit, 1, 5] = np.inf
    cache = make(hip_ctx, b, KVH, 64)
    with Device(hip_ctx) as dev:
        append(dev, cache, ref.whole(rng, b).on(dev), k, v, "f16")
        got = attend(dev, cache, b.on(dev), q, dtype)
        windowed = attend(dev, cache, b.on(dev), q, dtype, window=10)
    cache.close()
    bad = np.zeros(got.shape, bool)
    bad[hit - start:, 2:4] = True  # the queries of KV head 1 at and past the token
    assert np.array_equal(np.isnan(got), bad)
    bad[hit - start + 10:] = False  # and those whose window has left it
    assert np.array_equal(np.isnan(windowed), bad)
    some = [0, 2, 3, heads - 1]
    want, bound = ref.attention(q, *clean, start, dtype, 10, heads=some)
    near = np.abs(windowed.astype(np.float64) - want) <= bound
    assert near[:, some][~bad[:, some]].all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,tokens", [(4, 60), (64, 300)])
def test_positions_without_a_page(hip_ctx, heads, tokens, dtype):
    """A query that sees a page that there is not, or a position past the table, gets NaN; one of a negative position zeros."""
    rng = np.random.default_rng(14)
    b = Batch(rng, 16, [tokens, tokens, tokens, 1], [tokens + 40, tokens + 40, tokens // 2, 5], spare_rows=1)
    q = rows(rng, b.rows, heads, 64, dtype)
    cache = make(hip_ctx, b, heads, 64)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        broken = (40 + tokens // 2) // 16  # a page of the first sequence
        b.table[0, broken] = b.pages
        table = b.table
        cut = -(-(tokens + 40) // 16) - 2  # the second one's last positions, past the table
        b.table = np.ascontiguousarray(table[:, :cut])
        b.stride = cut
        got = attend(dev, cache, b.on(dev), q, dtype)
        windowed = attend(dev, cache, b.on(dev), q, dtype, window=16)
    cache.close()
    pos = np.arange(tokens) + 40
    gone = (pos >= broken * 16) | (pos >= cut * 16)
    assert np.array_equal(np.isnan(got[:tokens]).all((1, 2)), gone)
    assert np.isfinite(got[:tokens][~gone]).all()
    near = (pos >= broken * 16) & (pos < broken * 16 + 31) | (pos >= cut * 16)
    assert np.array_equal(np.isnan(windowed[:tokens]).all((1, 2)), near) and np.isfinite(windowed[:tokens][~near]).all()
    past = pos >= cut * 16
    assert np.array_equal(np.isnan(got[tokens:2 * tokens]).all((1, 2)), past)
    third = got[2 * tokens:3 * tokens]
    few = tokens - tokens // 2
    assert (third[:few] == 0).all()
    want, bound = ref.attention(q[2 * tokens + few:3 * tokens], *data[2], 0, dtype, heads=[0, heads - 1])
    assert (np.abs(third[few:].astype(np.float64) - want) <= bound)[:, [0, heads - 1]].all()
    want, bound = ref.attention(q[3 * tokens:3 * tokens + 1], *data[3], 4, dtype)
    assert (np.abs(got[3 * tokens:3 * tokens + 1].astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,new,n", [(4, 4, 3, 70), (64, 64, 300, 350), (16, 2, 300, 350)])
def test_the_table_ends_inside_a_step(hip_ctx, heads, kv_heads, new, n, dtype):
    """Queries past a table of an odd number of pages of 16 get NaN, those before it what they see; the other pages hold NaN."""
    rng = np.random.default_rng(31)
    b = Batch(rng, 16, [new], [n])
    q = rows(rng, new, heads, 64, dtype)
    cache = make(hip_ctx, b, kv_heads, 64)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        cut = n // 16 - 1 - (n // 16) % 2  # (odd: half a step)
        assert cut % 2 == 1 and cut * 16 > n - new or new == 3
        b.table, b.stride = np.ascontiguousarray(b.table[:, :cut]), cut
        for i in set(range(b.pages)) - set(b.table.ravel().tolist()):
            for buf in (cache._desc.k, cache._desc.v):
                size = cache.bytes // 2 // b.pages
                L.check(L.lib().ahip_memset(hip_ctx.handle, buf + i * size, 0xFF, size))
        # (page 0 stands in for one that there is not: NaN there too, where the sequence does not have it)
        got = attend(dev, cache, b.on(dev), q, dtype)
    cache.close()
    past = np.arange(n - new, n) >= cut * 16
    assert np.array_equal(np.isnan(got).all((1, 2)), past) and np.isfinite(got[~past]).all()
    if (~past).any():
        some = [0, heads - 1]
        want, bound = ref.attention(q, *data[0], n - new, dtype, heads=some)
        assert (np.abs(got.astype(np.float64) - want) <= bound)[:, some][~past].all()


@pytest.mark.parametrize("window", [0, 40, 2**30, 2**31 - 1])
@pytest.mark.parametrize("heads,rows_more", [(4, 5), (64, 200)])
def test_rows_of_negative_positions_beside_others(hip_ctx, heads, rows_more, window):
    """More rows than the length says: zeros for those, the others' attention as it is, under any window."""
    rng = np.random.default_rng(32)
    n = 60 if heads == 4 else 150
    b = Batch(rng, 16, [n + rows_more], [n])
    q = rows(rng, b.rows, heads, 64, "f32")
    cache = make(hip_ctx, b, heads, 64)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        got = attend(dev, cache, b.on(dev), q, "f32", window=window, sinks=window and 3)
    cache.close()
    assert (got[:rows_more] == 0).all()
    some = [0, heads - 1]
    want, bound = ref.attention(q[rows_more:], *data[0], 0, "f32", window, window and 3, heads=some)
    assert (np.abs(got[rows_more:].astype(np.float64) - want) <= bound)[:, some].all()


@pytest.mark.parametrize("heads,tokens", [(4, 3), (64, 300)])
def test_batches_that_say_too_much_stay_inside_their_arrays(hip_ctx, heads, tokens):
    """Row starts past the rows or falling, lengths below 0 and far past the table: no row outside the arrays is touched,
    and the sequences in order are what they are."""
    rng = np.random.default_rng(15)
    b = Batch(rng, 16, [tokens, 1], [tokens + 9, 50])
    q = rows(rng, b.rows, heads, 64, "f16")
    cache = make(hip_ctx, b, heads, 64)
    with Device(hip_ctx) as dev:
        data = fill(dev, cache, rng, b)
        for starts, lengths in (([0, tokens, 2**31 - 1], [tokens + 9, 50]), ([0, tokens, -5], [tokens + 9, 50]),
                                ([-(2**31), tokens, tokens + 1], [tokens + 9, -(2**31)]),
                                ([0, tokens, tokens + 1], [tokens + 9, 2**31 - 1])):
            on = PagedBatch(dev.put(np.array(starts, np.int32)), dev.put(np.array(lengths, np.int32)), dev.put(b.table), 2,
                            b.stride, b.rows, tokens)
            got = attend(dev, cache, on, q, "f16", extra=8)
            load(dev, cache, on, b.rows, "f16", extra=8)
            want, bound = ref.attention(q[:tokens], *data[0], 9, "f16", heads=[1])
            assert (np.abs(got[:tokens].astype(np.float64) - want) <= bound)[:, 1].all()
            if starts[2] == -5:
                assert untouched(got[tokens:])
            elif lengths[1] < 0:
                assert (got[tokens:] == 0).all()
            elif lengths[1] > 50:
                assert np.isnan(got[tokens:]).all()
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_shared_pages(hip_ctx, dtype):
    """Two conversations with one beginning: the same pages in both tables."""
    rng = np.random.default_rng(16)
    b = Batch(rng, 32, [1, 4], [200, 180])
    b.table[1, :3] = b.table[0, :3]
    cache = make(hip_ctx, b, 2, 64)
    q = rows(rng, b.rows, 6, 64, dtype)
    with Device(hip_ctx) as dev:
        for s in (1, 0):  # one after the other, so that the beginning is the first one's
            one = ref.whole(rng, b)
            one.new = [n if i == s else 0 for i, n in enumerate(one.lengths)]
            one.starts = [0, one.new[0], sum(one.new)]
            one.rows = sum(one.new)
            k, v = (rows(rng, one.rows, 2, 64, "f16") for _ in range(2))
            append(dev, cache, one.on(dev), k, v, "f16")
            if s == 1:
                second = k, v
        data = [(k, v), tuple(np.concatenate([x[:96], y[96:]]) for x, y in zip((k, v), second))]
        got = attend(dev, cache, b.on(dev), q, dtype)
    cache.close()
    check(got, q, data, b, dtype, "shared")


def test_attention_twice_gives_the_same_bits(hip_ctx):
    rng = np.random.default_rng(17)
    b = Batch(rng, 16, [1, 3, 200, 1], [5000, 3000, 900, 20])
    q = rows(rng, b.rows, 8, 128, "f32")
    cache = make(hip_ctx, b, 8, 128)
    with Device(hip_ctx) as dev:
        fill(dev, cache, rng, b)
        on = b.on(dev)
        a = attend(dev, cache, on, q, "f32")
        need = cache.workspace_bytes()
        mine = (dev.empty(need, 0xFF), need)  # another workspace, its bytes NaN but for the counters
        L.check(L.lib().ahip_memset(hip_ctx.handle, mine[0], 0, PAGED_WORKSPACE_ZERO))
        c = attend(dev, cache, on, q, "f32", workspace=mine)
        with pytest.raises(L.InvalidArgument, match="workspace"):
            attend(dev, cache, on, q, "f32", workspace=(mine[0], need - 1))
    cache.close()
    assert np.array_equal(a.view(np.uint32), c.view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_one_workspace_serves_turns_and_single_tokens_in_turn(hip_ctx, dtype):
    rng = np.random.default_rng(20)
    full = Batch(rng, 64, [0] * 3, [5000, 3000, 100])
    cache = make(hip_ctx, full, 8, 128)
    with Device(hip_ctx) as dev:
        fill(dev, cache, rng, full)
        need = cache.workspace_bytes()
        one = dev.empty(need, 0xFF)
        L.check(L.lib().ahip_memset(hip_ctx.handle, one, 0, PAGED_WORKSPACE_ZERO))
        for new, lengths in [([200], [5000]), ([1, 1], [5000, 2999]), ([150, 1, 1], [5000, 3000, 100]), ([200], [5000])] * 2:
            b = Batch(rng, 64, new, lengths, full.pages, stride=full.stride)
            b.table = full.table[:len(new)].copy()
            q = rows(rng, b.rows, 32, 128, dtype)
            a = attend(dev, cache, b.on(dev), q, dtype, workspace=(one, need))
            c = attend(dev, cache, b.on(dev), q, dtype)
            assert np.isfinite(a).all() and np.array_equal(a.view(np.uint8), c.view(np.uint8)), (new, lengths)
            assert not dev.get(one, PAGED_WORKSPACE_ZERO, np.uint8).any()
    cache.close()


def test_one_workspace_serves_batches_of_every_shape_in_turn(hip_ctx):
    rng = np.random.default_rng(18)
    shapes = [([1], [6000]), ([1] * 40, [150 * i + 1 for i in range(40)]), ([500, 1], [2000, 5000]), ([3], [3]),
              ([20, 1, 1], [4000, 6000, 10]), ([1], [6000])] * 2
    full = Batch(rng, 64, [0] * 40, [6000] * 40)
    cache = make(hip_ctx, full, 8, 64)
    with Device(hip_ctx) as dev:
        fill(dev, cache, rng, full)
        need = cache.workspace_bytes()
        one = dev.empty(need)
        L.check(L.lib().ahip_memset(hip_ctx.handle, one, 0, PAGED_WORKSPACE_ZERO))
        for new, lengths in shapes:
            b = Batch(rng, 64, new, lengths, full.pages, stride=full.stride)
            b.table = full.table[:len(new)].copy()
            q = rows(rng, b.rows, 16, 64, "f32")
            a = attend(dev, cache, b.on(dev), q, "f32", workspace=(one, need))
            c = attend(dev, cache, b.on(dev), q, "f32")
            assert np.isfinite(a).all() and np.array_equal(a.view(np.uint32), c.view(np.uint32)), (new, lengths)
            assert not dev.get(one, PAGED_WORKSPACE_ZERO, np.uint8).any()
    cache.close()


def test_two_streams_with_workspaces_of_their_own(hip_ctx):
    rng = np.random.default_rng(19)
    b = Batch(rng, 32, [1, 1], [7000, 400])
    cache = make(hip_ctx, b, 3, 64)
    streams = [C.c_void_p() for _ in range(2)]
    for s in streams:
        L.check(L.lib().ahip_stream_create(hip_ctx.handle, C.byref(s)))
    with Device(hip_ctx) as dev:
        fill(dev, cache, rng, b)
        on, need = b.on(dev), cache.workspace_bytes()
        qs = [rows(rng, 2, 12, 64, "f32") for _ in streams]
        want = [attend(dev, cache, on, q, "f32") for q in qs]
        ws, outs = [(dev.empty(need, 0), need) for _ in streams], [dev.empty(2 * 12 * 64 * 4) for _ in streams]
        qp = [dev.put(q) for q in qs]
        for _ in range(50):
            for s, w, o, q in zip(streams, ws, outs, qp):
                cache.attention(on, q, o, 12, workspace=w, stream=s)
        for s in streams:
            L.check(L.lib().ahip_stream_synchronize(s))
        for o, w in zip(outs, want):
            assert np.array_equal(dev.get(o, w.shape, np.float32).view(np.uint32), w.view(np.uint32))
    for s in streams:
        L.check(L.lib().ahip_stream_destroy(s))
    cache.close()


def test_an_empty_batch_does_nothing(hip_ctx):
    rng = np.random.default_rng(20)
    b = Batch(rng, 16, [0, 0], [5, 0], spare_rows=3)
    cache = make(hip_ctx, b, 2, 64)
    with Device(hip_ctx) as dev:
        q = rows(rng, 3, 4, 64, "f32")
        assert untouched(attend(dev, cache, b.on(dev), q, "f32"))
        append(dev, cache, b.on(dev), q[:, :2], q[:, 2:], "f32")
        assert (dev.get(cache._desc.k, cache.bytes // 2, np.uint8) == 0xFF).all()
        assert all(untouched(x) for x in load(dev, cache, b.on(dev), 3, "f32"))
    cache.close()
