"""Calls of mxfp4_grouped_gemm by the kernel that they are for: a test on the GPU compares their results
and one without a GPU asserts, by launches, that each still takes the kernel named here."""
from __future__ import annotations

# (dtype of the results, gated, activation)
FORMS = [("f32", False, "silu"), ("bf16", False, "silu"), ("f16", False, "silu"),
         ("f32", True, "gelu"), ("bf16", True, "silu"), ("f16", True, "gelu")]

# Rows of an expert around the heights of 32-row fragments and of tiles of 128 rows.
AROUND_128 = [1, 0, 127, 128, 129, 64, 65, 63, 33, 2]
# ... and of tiles of 256.
AROUND_256 = [300, 0, 257, 513, 129, 256, 65, 1]

# (rows of every expert, K, N, rows of a tile). Two rows behind the last expert's go along.
TILES = [
    # one block to many slices, the last of them whole and partial; odd widths
    (AROUND_128, 20, 1001, 128),
    (AROUND_128, 256, 1024, 128),
    (AROUND_128, 300, 1003, 128),
    (AROUND_128, 1023, 999, 128),
    (AROUND_128, 2337, 902, 128),
    ([126] + [128] * 7, 520, 1100, 128),  # the most rows an expert
    # several rounds of tiles: the last one cut; with short tiles that begin in a whole round
    ([100] * 20, 96, 4500, 128),
    ([128] * 10 + [100] * 9 + [98], 64, 6500, 128),
    ([44] * 596, 40, 33, 128),  # the most experts whose bounds three stages leave LDS for
    ([44] * 597, 40, 33, 256),
    ([20] * 500 + [0] * 24 + [100] * 500, 70, 37, 256),
    (AROUND_256, 20, 1001, 256),
    (AROUND_256, 256, 768, 256),
    (AROUND_256, 300, 1003, 256),
    (AROUND_256, 1023, 999, 256),
    (AROUND_256, 2337, 578, 256),
    ([128] * 7 + [127], 520, 1100, 256),  # one row more than tiles of 128 take
    ([2000, 0, 300], 96, 9001, 256),
    ([256] * 5 + [456] * 5, 64, 8960, 256),
]

# Rows of a tile: rows an expert and columns of the products with scales far apart and with offsets that do not
# rise (K = 320, three experts and more).
TILE_SIZES = {128: (100, 2050), 256: (300, 2050)}

# The kernel for few rows: (rows of every expert, K, N of plain and of gated products, [waves, weight rows of a
# workgroup, 1 where the weights are loaded past the caches]).
FEW_ROWS = [
    ([20, 3], 4100, 500, 251, [8, 32, 0]),
    ([20, 3], 1100, 300, 149, [4, 32, 0]),
    ([20, 3], 4100, 5501, 2751, [8, 64, 0]),
    ([20, 3], 2100, 6001, 3001, [4, 64, 0]),
    ([20, 3], 600, 101, 130, [2, 64, 0]),
    ([7, 0, 33], 200, 97, 64, [1, 64, 0]),
    ([7], 20000, 8001, 4001, [8, 32, 1]),
    ([7, 8], 9000, 8201, 4101, [8, 64, 1]),
    ([7, 8, 6, 5], 4200, 8201, 4101, [4, 64, 1]),
    ([3] * 31 + [1], 600, 7001, 3501, [2, 64, 1]),
    ([2] * 63 + [1], 200, 9401, 4701, [1, 64, 1]),
]
