"""Sizes of sort_tokens, combine_tokens and their gradients that take every kernel of theirs, for tests on the GPU and
for one that asserts by launches that none is left out."""
from __future__ import annotations

# types of the sorted rows and of the tokens' rows
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]


def width(dtype, pieces, whole):
    """Columns of a row of so many pieces of 16 bytes, the last of them whole or one column short."""
    return pieces * (4 if dtype == "f32" else 8) - (0 if whole else 1)


# Pieces of a row for every number of threads a token: 8, 16, 32, 64, 128 and 256.
PIECES = [5, 12, 30, 50, 100, 200]

# (tokens, top_k, experts, pieces, whole)
SORT = (
    [(9, 3, 7, 5, True)]
    # one launch: rows of any width, of whole pieces, and past the caches
    + [(700, 3, experts, 30, whole) for experts in (9, 300) for whole in (True, False)]
    + [(3001, 2, experts, 180, True) for experts in (9, 300)]
    # the rows in a launch of their own, up to 64 threads a token in the caches and past them
    + [(8300, 2, 9, pieces, whole) for pieces in PIECES for whole in (True, False)]
    + [(11000, 2, 300, 50, True)]
)
MAPS = [(9, 3, 7), (700, 3, 9), (700, 3, 300), (8300, 2, 9), (8300, 2, 300)]

# (tokens, top_k, pieces, whole): four and eight routes together; two pieces a thread; results past the caches
COMBINE = (
    [(70, top_k, pieces, whole) for pieces in PIECES for top_k in (3, 9) for whole in (True, False)]
    + [(1030, top_k, 300, whole) for top_k in (3, 9) for whole in (True, False)]
    + [((1 << 20) // pieces + 1, top_k, pieces, True) for pieces in (50, 100, 200, 300) for top_k in (1, 5)]
)

# (rows, hidden) of quantize_rows_mxfp4: 32, 64 and 256 threads a row, a wave of many rows; whole pieces and not
QUANTIZE = [(300, 256), (300, 251), (300, 512), (300, 509), (40, 2048), (40, 2041), (1030, 600), (1030, 601)]
