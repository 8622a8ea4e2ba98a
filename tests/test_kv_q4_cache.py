"""Q4Cache's buffers where an allocation fails or the context is closed first,
on a stand-in for the library's allocator: no device, so on the CPU."""
import ctypes as C

import pytest

from alpaca_amd import _lib as L
from alpaca_amd.model import HIPContext
from alpaca_amd.kvcache import Q4Cache


class Allocator:
    """The library's calls that a cache makes, over addresses that it counts: `fails` the allocations (from 1) that
    are refused.  Everything else is the library's own."""

    def __init__(self, fails):
        self.fails, self.calls, self.held, self.contexts = set(fails), 0, {}, 0

    def ahip_malloc(self, ctx, n, out):
        self.calls += 1
        assert ctx
        if self.calls in self.fails:
            return L.ALLOC
        p = self.calls << 20
        self.held[p] = n
        C.cast(out, C.POINTER(C.c_void_p))[0] = p
        return 0

    def ahip_free(self, ctx, p):
        assert ctx
        del self.held[p]  # (freed once)
        return 0

    def ahip_memset(self, ctx, p, value, n):
        assert p in self.held
        return 0

    def ahip_attention_q4_workspace(self, ctx, cache, dtype, tokens, heads, start, on_device, n):
        if not ctx:
            return L.INVALID_ARGUMENT
        C.cast(n, C.POINTER(C.c_int64))[0] = 4096 * tokens
        return 0

    def ahip_attention_q4(self, ctx, cache, dtype, q, qs, tokens, heads, start, start_dev, out, os, work, n, stream):
        if not ctx:
            return L.INVALID_ARGUMENT
        assert n >= 4096 * tokens and work in self.held
        return 0

    def ahip_context_destroy(self, ctx):
        self.contexts += 1
        return 0

    def __getattr__(self, name):
        return getattr(self.real, name)


@pytest.fixture
def made(monkeypatch):
    """make(fails) -> (allocator, context), the allocator in the library's place from then on."""
    real, contexts = L.lib(), []

    def make(fails=()):
        a = Allocator(fails)
        a.real = real
        monkeypatch.setattr(L, "lib", lambda: a)
        c = HIPContext.__new__(HIPContext)
        c.handle, c.device, c._kind = C.c_void_p(1 << 20), 0, "context"
        contexts.append(c)
        return a, c
    yield make
    for c in contexts:
        c.close()


@pytest.mark.parametrize("fails", [1, 2])
def test_a_cache_that_cannot_be_allocated_keeps_nothing(made, fails):
    a, ctx = made([fails])
    with pytest.raises(L.HIPError) as e:
        Q4Cache(ctx, 2, 64, 64)
    assert e.value.code == L.ALLOC and not a.held
    cache = Q4Cache(ctx, 2, 64, 64)  # the next one is whole
    assert len(a.held) == 2
    cache.close()
    assert not a.held


def test_a_workspace_that_cannot_grow_is_allocated_by_the_next_call(made):
    a, ctx = made([4])
    cache = Q4Cache(ctx, 2, 64, 64)
    cache.attention(1 << 10, 1 << 12, 1, 4)
    with pytest.raises(L.HIPError):
        cache.attention(1 << 10, 1 << 12, 8, 4)
    cache.attention(1 << 10, 1 << 12, 1, 4)  # a shape that ran before
    cache.attention(1 << 10, 1 << 12, 8, 4)
    assert sorted(a.held.values())[-1] == 8 * 4096 and len(a.held) == 3
    cache.close()
    assert not a.held


def test_a_closed_context_frees_its_caches_and_refuses_their_calls(made):
    _, ctx = made()
    b, other = made()
    caches = [Q4Cache(other, 2, 64, 64) for _ in range(2)]
    caches[0].attention(1 << 10, 1 << 12, 1, 4)
    assert len(b.held) == 5
    ctx.close()
    assert len(b.held) == 5  # another context's
    other.close()
    assert not b.held and b.contexts == 2
    for cache in caches:
        for call in (lambda: cache.store(1 << 10, 1 << 10, 1), lambda: cache.load(1 << 10, None, 1),
                     lambda: cache.attention(1 << 10, 1 << 12, 1, 4),
                     lambda: cache.attention(1 << 10, 1 << 12, 1, 4, workspace=(1 << 20, 1 << 20)),
                     lambda: cache.workspace_bytes(1, 4)):
            with pytest.raises(L.InvalidArgument):
                call()
        cache.close()  # (again: nothing)


def test_a_closed_cache_refuses_its_calls(made):
    a, ctx = made()
    cache = Q4Cache(ctx, 2, 64, 64)
    cache.close()
    assert not a.held
    for call in (lambda: cache.store(1 << 10, 1 << 10, 1), lambda: cache.load(1 << 10, None, 1)):
        with pytest.raises(L.InvalidArgument):
            call()
