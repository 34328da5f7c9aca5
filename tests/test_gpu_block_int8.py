"""quantize_rows and int8_grouped_gemm against their definitions.

quantize_rows is exact (two FP32 divisions and a rounding to even). Sums of int8
products are exact, so y is off by FP32 roundings only: of the sum, the two scales'
products (four half units) and the output type; the gated form by 2^-20 for the
exponential on top, and by the preactivation's error (four half units of FP32 times
|p| act'/act <= |p| + 1).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_amd as rr
from block_helpers import ACTIVATIONS, CODES, LEAST, ROUNDING, TYPES, Buf, assert_within, context, offsets_of, segments

pytestmark = pytest.mark.gpu
FAMILIES = {"auto": rr.kernel(), "naive": rr.kernel(rr.KernelFamily.kNaive)}


def quantize(x, dtype, offset=0):
    rows, hidden = x.shape
    q, s = Buf(shape=(rows, hidden), dtype=torch.int8, offset=offset), Buf(shape=(rows,), dtype=torch.float32)
    xb = Buf(x, offset=offset)
    ctx, _ = context()
    status = rr.quantize_rows(rr.QuantizeRowsArgs(x=xb.ptr, q=q.ptr, scale=s.ptr, rows=rows, hidden=hidden,
                                                  dtype=CODES[dtype]), ctx)
    assert status.ok(), status.message
    assert q.intact() and s.intact() and xb.intact()
    return q, s


@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (5, 512), (2, 513), (7, 1000), (4, 1024), (3, 2047),
                                         (2, 4096), (2, 8190), (2, 16384), (2, 20001), (300, 264)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset", [0, 3])
def test_quantize_rows(device, rows, hidden, dtype, offset):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(rows * hidden)
    x = torch.randn(rows, hidden, device="cuda:0", generator=gen)
    x *= torch.logspace(-3, 3, rows, device="cuda:0")[:, None]
    x[0] = 0.0 if rows > 1 else x[0]
    x = x.to(TYPES[dtype])
    q, s = quantize(x, dtype, offset)
    host = x.float().cpu().numpy()
    scale = (np.abs(host).max(axis=1) / np.float32(127.0)).astype(np.float32)
    with np.errstate(invalid="ignore", divide="ignore"):
        want = np.where(scale[:, None] > 0, np.rint(host / scale[:, None]), 0).astype(np.int8)
    assert np.array_equal(s.t.cpu().numpy(), scale)
    assert np.array_equal(q.t.cpu().numpy(), want)


def test_quantize_rows_special_values(device):
    x = torch.ones(5, 40, device="cuda:0")
    x[1, 3], x[2, 39], x[3, 0] = float("inf"), float("nan"), float("-inf")
    x[4] = 1e-45  # a scale below the least FP32 number
    q, s = quantize(x, "f32")
    s, q = s.t.cpu(), q.t.cpu()
    assert s[1] == float("inf") and torch.isnan(s[2]) and s[3] == float("inf") and s[4] == 0
    assert (q[0] == 127).all() and (q[1:] == 0).all()


def product(q, qs, weights, scales, counts, n, dtype, act, family, offset=0):
    rows, k = q.shape
    bufs = [Buf(t, offset=o) for t, o in ((q, offset), (qs, 0), (weights[0], offset), (scales[0], 0))]
    gated = len(weights) == 2
    up = [Buf(weights[1], offset=offset), Buf(scales[1])] if gated else []
    offs = Buf(offsets_of(counts)[0])
    y = Buf(shape=(rows, n), dtype=TYPES[dtype], offset=offset)
    args = rr.Int8GroupedGemmArgs(q=bufs[0].ptr, q_scale=bufs[1].ptr, w=bufs[2].ptr, w_scale=bufs[3].ptr,
                                  w_up=up[0].ptr if gated else None, w_up_scale=up[1].ptr if gated else None,
                                  offsets=offs.ptr, y=y.ptr, rows=rows, experts=len(counts), hidden=k, output=n,
                                  activation=int(ACTIVATIONS[act][0]), dtype=CODES[dtype], kernel=FAMILIES[family])
    ctx, ws = context(rr.get_int8_grouped_gemm_workspace_size(args))
    status = rr.int8_grouped_gemm(args, ctx)
    assert status.ok(), status.message
    for buf in (*bufs, *up, offs, y, ws):
        assert buf.intact()
    return y


SHAPES = [
    ([1], 1, 1),
    ([2, 0, 1], 16, 3),
    ([0, 5, 0, 17, 1, 0], 33, 47),
    ([16, 15], 64, 64),
    ([0, 3], 256, 128),
    ([1, 1, 0, 6], 512, 272),
    ([70, 0, 31], 144, 200),
    ([129, 64, 1], 257, 130),
    ([256, 300], 128, 264),
    ([600, 9], 1040, 512),
    ([0, 37, 0, 1, 2] + [0] * 9, 272, 96),
]


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("dtype,gated,act", [("f32", False, "silu"), ("bf16", True, "silu"), ("f16", True, "gelu"),
                                             ("bf16", False, "silu")])
@pytest.mark.parametrize("counts,k,n", SHAPES)
def test_products(device, counts, k, n, dtype, gated, act, family):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(k * n)
    offs, rows = offsets_of(counts)
    e = len(counts)
    q = torch.randint(-127, 128, (rows, k), device="cuda:0", generator=gen, dtype=torch.int8)
    qs = torch.rand(rows, device="cuda:0", generator=gen) * 0.02 + 0.001
    weights = [torch.randint(-127, 128, (e, n, k), device="cuda:0", generator=gen, dtype=torch.int8)
               for _ in range(1 + gated)]
    scales = [(torch.rand(e, n, device="cuda:0", generator=gen) + 0.1) * 0.02 * k ** -0.5 for _ in weights]
    for offset in (0, 1):
        y = product(q, qs, weights, scales, counts, n, dtype, act, family, offset).t
        u, least, f32 = ROUNDING[dtype], LEAST[dtype], 4 * ROUNDING["f32"]
        for x, seg in segments(counts):
            p = [(q[seg].double() @ w[x].double().t().contiguous()) * qs[seg, None].double() * s[x].double()
                 for w, s in zip(weights, scales)]
            if gated:
                a = ACTIVATIONS[act][1](p[0])
                want = a * p[1]
                # act's own error: 2^-20 of it, and 1.2 |p| of the preactivation's
                bound = (want.abs() * (2.0 ** -20 + f32) + 1.2 * p[0].abs() * f32 * p[1].abs()) * (1 + u) + u * want.abs()
            else:
                want = p[0]
                bound = want.abs() * (u + f32 * (1 + u))
            assert_within(y[seg], want, bound + least, f"y of expert {x}")


@pytest.mark.parametrize("family", ["auto", "naive"])
def test_extremes_and_rows_past_the_last(device, family):
    """All products of one sign at the largest magnitude, an expert without rows, and rows
    past the segments left alone."""
    counts, k, n = [3, 0, 2], 4096, 40
    q = torch.full((7, k), -128, dtype=torch.int8, device="cuda:0")
    w = torch.full((3, n, k), -128, dtype=torch.int8, device="cuda:0")
    qs, ws = torch.ones(7, device="cuda:0"), torch.ones(3, n, device="cuda:0")
    qs[1] = float("nan")
    y = product(q, qs, [w], [ws], counts, n, "f32", "silu", family)
    t = y.t
    assert torch.isnan(t[1]).all()
    assert (t[[0, 2, 3, 4]] == 128.0 * 128.0 * k).all()
    assert y.untouched(slice(5, None))


def test_neighbours_do_not_leak(device):
    """The rows and channels next to a ragged tile do not enter it."""
    counts, k, n = [5, 130], 72, 72
    q = torch.full((135, k), 1, dtype=torch.int8, device="cuda:0")
    w = torch.full((2, n, k), 1, dtype=torch.int8, device="cuda:0")
    w[1] = 100
    qs, ws = torch.ones(135, device="cuda:0"), torch.ones(2, n, device="cuda:0")
    t = product(q, qs, [w], [ws], counts, n, "f32", "silu", "auto").t
    assert (t[:5] == k).all() and (t[5:] == 100 * k).all()
