"""The shapes that the GPU tests of the attention over pages are to reach every kernel with."""
import random

from tests.paged_shapes import BOTH, BUILT, SHAPES, variant


def test_every_kernel_has_a_shape():
    reached = set()
    for hd, v, (heads, kv_heads, page, new, lengths, types) in SHAPES:
        for d in types:
            positions = max(-(-n // page) for n in lengths) * page
            for spare in (0, 2):  # (the GPU tests' batches have two rows of no sequence)
                assert variant(hd, d, heads, kv_heads, len(new), sum(new) + spare, max(new), 0, positions) == v, (hd, v, d, new)
            reached.add((hd, v, d))
    assert reached == BUILT


def test_no_call_needs_another():
    rng = random.Random(1)
    for _ in range(20000):
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 16, 32, 64, 96])
        sequences, most, hd, d = rng.choice([1, 1, 2, 5, 32]), rng.randint(1, 6000), 32 * rng.randint(1, 8), rng.choice(BOTH)
        v = variant(hd, d, kv_heads * rng.choice([1, 2, 3, 5, 8]), kv_heads, sequences, most + sequences - 1, most, 0,
                    rng.choice([500, 4096]))
        assert v is None or (hd, v, d) in BUILT
