"""Which kernel a 4-bit product takes, by the launches that a stand-in for HIP sees (no GPU is used). The
tests on the GPU take their cases from the same lists, so that a rule that sends them elsewhere fails here."""
from __future__ import annotations

import re

from block_helpers import CODES
from mxfp4_cases import FEW_ROWS, FORMS, TILE_SIZES, TILES
from stand_in import P, launched
from test_gpu_block_offsets import OFFSETS


def product(rows, experts, k, n, dtype, gated):
    up = dict(w_up=P, w_up_scale=P) if gated else {}
    return ["mxfp4_grouped_gemm", dict(q=P, q_scale=P, w=P, w_scale=P, offsets=P, y=P, rows=rows, experts=experts, hidden=k,
                                       output=n, dtype=CODES[dtype], **up)]


def same_kernels(folder, cases):
    """cases: (call, [rows of a tile] or the kernel for few rows' [waves, weight rows, past the caches])."""
    wrong = []
    for (call, want), names in zip(cases, launched(folder, [call for call, _ in cases])[0]):
        assert len(names) == 1
        tile = re.search(r"rr_mxfp4_gemm_kernel.*Li(\d+)E", names[0])
        few = re.search(r"rr_mxfp4_rows_kernel.*Li(\d+)ELi(\d+)ELb(\d)E", names[0])
        got = [int(v) for v in (tile or few).groups()]
        if got != want:
            wrong.append((call, got, want))
    assert not wrong


def test_tiles(tmp_path):
    same_kernels(tmp_path, [(product(sum(counts) + 2, len(counts), k, n, dtype, gated), [tile])
                            for counts, k, n, tile in TILES for dtype, gated, _ in FORMS])


def test_tiles_of_special_cases(tmp_path):
    same_kernels(tmp_path, [(product(experts * rows, experts, k, n, dtype, gated), [tile])
                            for tile, (rows, n) in TILE_SIZES.items()
                            for experts in [len(o) - 1 for o in OFFSETS.values()] + [4]
                            for k in (72, 320) for dtype in ("f32", "bf16") for gated in (False, True)])


def test_few_rows(tmp_path):
    same_kernels(tmp_path, [(product(sum(counts) + 2, len(counts), k, n_gated if gated else n, dtype, gated), kernel)
                            for counts, k, n, n_gated, kernel in FEW_ROWS for dtype, gated, _ in FORMS])
