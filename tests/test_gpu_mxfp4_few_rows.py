"""mxfp4_grouped_gemm on every form of its kernel for few rows, in every type of results, plain and gated;
test_mxfp4_kernels.py asserts that these cases are that kernel's. Bounds as in test_gpu_mxfp4_tiles.py."""
from __future__ import annotations

import pytest
import torch

from mxfp4_cases import FEW_ROWS, FORMS
from test_gpu_mxfp4_tiles import case, check, multiply

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,gated,act", FORMS)
@pytest.mark.parametrize("index", range(len(FEW_ROWS)), ids=lambda i: f"{FEW_ROWS[i][1]}-{FEW_ROWS[i][4]}".replace(", ", "-"))
def test_products(device, index, dtype, gated, act):
    counts, k, n, n_gated, _ = FEW_ROWS[index]
    n = n_gated if gated else n
    x, parts, offsets = case(counts, k, n, gated, index)
    y = multiply(x, parts, offsets, n, dtype, act)
    # (large weights: the first and the last channels, which end inside a workgroup's, and some between)
    columns = None
    if n * len(counts) * k > 1 << 24:
        columns = torch.cat([torch.arange(70), torch.arange(70, n - 70, 37), torch.arange(n - 70, n)]).cuda()
    check(y, x, parts, offsets, n, dtype, act, columns)
