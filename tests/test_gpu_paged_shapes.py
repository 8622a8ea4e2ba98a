"""Attention over pages on every kernel that is built for many columns (tests/paged_shapes.py says which a shape runs on)."""
import pytest

from tests.paged_shapes import SHAPES
from tests.test_gpu_paged import attention_case

pytestmark = pytest.mark.gpu

CASES = [(hd, v, dtype, *rest) for hd, v, (*rest, types) in SHAPES for dtype in types]


@pytest.mark.parametrize("hd,kernel,dtype,heads,kv_heads,page,new,lengths", CASES)
def test_attention_on_every_kernel(hip_ctx, hd, kernel, dtype, heads, kv_heads, page, new, lengths):
    some = [0, heads // 2, heads - 1]
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, some_heads=some)
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, extra=3, lead=1, some_heads=some, seed=1)


@pytest.mark.parametrize("hd,kernel,dtype,heads,kv_heads,page,new,lengths", [c for c in CASES if c[1] != (8, 1)])
def test_windows_on_every_kernel(hip_ctx, hd, kernel, dtype, heads, kv_heads, page, new, lengths):
    attention_case(hip_ctx, heads, kv_heads, hd, page, new, lengths, dtype, window=90, sinks=5,
                   some_heads=[0, heads // 2, heads - 1])
