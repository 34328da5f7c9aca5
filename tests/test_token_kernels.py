"""Every kernel of the operators that take tokens to their experts and back and of the 4-bit operators is one that the
tests on the GPU run, by the launches that a stand-in for HIP sees (no GPU is used)."""
from __future__ import annotations

import re

import raggedroute_amd as rr
from block_helpers import CODES
from mxfp4_cases import FEW_ROWS, FORMS, TILES
from stand_in import P, launched
from test_mxfp4_kernels import product
from token_cases import COMBINE, MAPS, PAIRS, QUANTIZE, SORT, width

KERNELS = re.compile(r"rr_(sort|combine|gate_backward|quantize_mxfp4|mxfp4)_")


def calls():
    for dtype, other in PAIRS:
        types = dict(dtype=CODES[dtype])
        maps = dict(x=P, expert_ids=P, offsets=P, route_pos=P, sorted_route=P, x_dtype=CODES[other], **types)
        for tokens, top_k, experts in MAPS:
            yield "sort_tokens", dict(tokens=tokens, top_k=top_k, experts=experts, hidden=8, **maps)
        for tokens, top_k, experts, pieces, whole in SORT:
            yield "sort_tokens", dict(x_sorted=P, tokens=tokens, top_k=top_k, experts=experts,
                                      hidden=width(dtype, pieces, whole), **maps)
        for tokens, top_k, pieces, whole in COMBINE:
            size = dict(tokens=tokens, top_k=top_k, hidden=width(dtype, pieces, whole), route_pos=P, **types)
            yield "sort_tokens_backward", dict(dx_sorted=P, dx=P, x_dtype=CODES[other], **size)
            size |= dict(y_sorted=P, route_weights=P, y_dtype=CODES[other])
            yield "combine_tokens", dict(y=P, **size)
            yield "combine_tokens_backward", dict(dy=P, dy_sorted=P, droute_weights=P, **size)
    yield "topk_gate_backward", dict(expert_ids=P, weights=P, dweights=P, dlogits=P, tokens=5, experts=9)
    for dtype in CODES:
        for rows, hidden in QUANTIZE:
            yield "quantize_rows_mxfp4", dict(x=P, q=P, scale=P, rows=rows, hidden=hidden, dtype=CODES[dtype])
    for dtype, gated, _ in FORMS:
        for counts, k, n, _ in TILES:
            yield product(sum(counts) + 2, len(counts), k, n, dtype, gated)
        for counts, k, n, n_gated, _ in FEW_ROWS:
            yield product(sum(counts) + 2, len(counts), k, n_gated if gated else n, dtype, gated)
    entry, fields = product(1, 1, 1, 1, "f32", False)
    yield entry, fields | dict(kernel=int(rr.KernelFamily.kNaive))


def test_every_kernel_is_called(tmp_path):
    runs, names = launched(tmp_path, list(calls()))
    ours = {name for name in names if KERNELS.search(name)}
    assert len(ours) > 100
    unused = ours - {name for run in runs for name in run}
    assert not unused, "\n".join(sorted(unused))
