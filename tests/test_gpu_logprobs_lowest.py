"""Log probabilities and entropies of rows whose masked logits are large negative numbers rather than -inf."""
import numpy as np
import pytest

from tests.paged_reference import NP
from tests.test_gpu_logprobs import check

pytestmark = pytest.mark.gpu

LOWEST = {"f32": [np.finfo(np.float32).min, -1e38, -3e37, -1e5], "f16": [np.finfo(np.float16).min, -6e4]}


def rows_of(vocab, value):
    """Few tokens that are allowed, at the ends, in one place or spread; masked ones before and behind them."""
    places = [[0], [vocab - 1], [vocab // 2], [0, vocab - 1], list(range(vocab // 2, min(vocab, vocab // 2 + 3))),
              list(range(1, vocab, max(1, vocab // 7)))]
    x = np.full((len(places) + 2, vocab), value, np.float64)
    for r, p in zip(x, places):
        r[p] = np.arange(len(p)) % 3 + 0.5
    x[-1] = np.where(np.arange(vocab) % 2, value, np.sin(np.arange(vocab)))  # (x[-2]: all masked, all alike)
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [2, 40, 3001, 49152, 100000])
@pytest.mark.parametrize("top", [0, 2])
def test_masks_of_the_type_s_lowest_values(hip_ctx, vocab, top, dtype):
    for value in LOWEST[dtype]:
        x = rows_of(vocab, value).astype(NP[dtype])
        tokens = np.arange(len(x)) * (vocab // 3) % vocab
        got = check(hip_ctx, x, tokens, top)  # (rows split over workgroups, where they are long)
        assert np.isfinite(got[1]).all()
        check(hip_ctx, x, tokens, top, workspace=(None, 0))
        check(hip_ctx, x, tokens, top, extra=5, lead=3)


def test_many_rows_of_the_lowest_value(hip_ctx):
    x = np.concatenate([rows_of(7000, v) for v in LOWEST["f32"]] * 20).astype(np.float32)
    check(hip_ctx, x, np.arange(len(x)) * 7 % 7000, 10, extra=3)
