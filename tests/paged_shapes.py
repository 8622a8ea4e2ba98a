"""Which kernel a call of the attention over pages runs, and shapes that reach every one of them."""

CUS = 256

# (head dim, (columns of a workgroup / 32, sets of waves)): (heads, kv_heads, page, new, lengths, types)
BOTH = ("f32", "f16")
SHAPES = [
    (32, (4, 2), (64, 64, 16, [300, 1], [333, 70], BOTH)),
    (32, (4, 1), (128, 64, 64, [300, 3], [310, 3], BOTH)),
    (64, (2, 4), (64, 64, 16, [250, 1], [777, 90], BOTH)),
    (64, (2, 4), (9, 3, 32, [1501], [1600], BOTH)),
    (64, (4, 2), (64, 64, 32, [290], [301], BOTH)),
    (64, (4, 1), (64, 64, 32, [650, 2, 1], [700, 9, 301], BOTH)),
    (96, (2, 4), (40, 40, 16, [250], [261], BOTH)),
    (96, (2, 4), (24, 8, 32, [300, 1], [2300, 77], BOTH)),
    (96, (4, 2), (64, 64, 64, [300], [450], BOTH)),
    (96, (4, 1), (64, 64, 16, [700], [701], BOTH)),
    (96, (8, 1), (64, 64, 16, [1700], [1733], BOTH)),
    (128, (2, 4), (32, 32, 16, [250, 4], [261, 31], BOTH)),
    (128, (4, 2), (64, 64, 16, [300], [450], BOTH)),
    (128, (4, 1), (64, 64, 32, [700], [701], BOTH)),
    (128, (8, 1), (64, 64, 32, [1601], [1601], BOTH)),
    (128, (8, 1), (32, 8, 64, [3500], [3529], BOTH)),
    (160, (4, 2), (64, 64, 32, [300], [350], ("f16",))),
    (160, (4, 1), (64, 64, 32, [300], [350], ("f32",))),
    (160, (4, 1), (64, 64, 32, [600, 1], [650, 3], ("f16",))),
    (192, (4, 2), (64, 64, 16, [257], [257], ("f16",))),
    (192, (4, 1), (64, 64, 16, [257], [257], ("f32",))),
    (192, (4, 1), (64, 64, 16, [600], [650], ("f16",))),
    (224, (4, 1), (64, 64, 32, [300], [350], BOTH)),
    (256, (4, 1), (64, 64, 32, [300], [350], BOTH)),
]


def variant(hd, dtype, heads, kv_heads, sequences, rows, max_rows, window, positions):
    """The rules of the attention's launch, at 256 CUs; None: sequences of few columns alone."""
    nb, group = hd // 32, heads // kv_heads
    max_rows = min(max_rows, rows) if max_rows else rows
    two = nb <= (4 if dtype == "f32" else 6)  # waves of a SIMD

    def groups(width):
        return -(-rows * group // width) * kv_heads
    if max_rows * group <= 64:
        return None
    more = max(1, max_rows - 1)
    single = sequences - (rows - sequences + more - 1) // more
    if nb in (3, 4) and sequences == 1 and not window and 5 * CUS <= 3 * groups(256) and groups(256) <= 2 * CUS:
        return 8, 1
    if groups(128) > CUS or groups(64) * nb > 8 * CUS // 5 and (not two or single * kv_heads >= 4 * groups(128)):
        return 4, 1
    if two and groups(64) > CUS:
        return 4, 2
    if 2 <= nb <= 4 and 10 * groups(64) * nb >= (11 if nb >= 3 and positions >= 2048 else 16) * CUS:
        return 2, 4
    return None


# every kernel for many columns that is built
BUILT = {(hd, v, d) for hd in range(32, 257, 32) for v in ((4, 1), (4, 2), (2, 4), (8, 1)) for d in BOTH
         if v == (4, 1) or v == (4, 2) and hd <= (128 if d == "f32" else 192) or v == (2, 4) and 64 <= hd <= 128
         or v == (8, 1) and hd in (96, 128)}
