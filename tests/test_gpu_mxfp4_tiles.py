"""mxfp4_grouped_gemm on its tile kernels, in every type of results, plain and gated, against the
definition in 64 bits; test_mxfp4_kernels.py asserts that these cases are the tile kernels'.

A term of a sum is exact, a sum over K elements takes K roundings to FP32 at most of partial sums no larger than the
sum of the terms' magnitudes, and a result is rounded to its type. The gated form adds 2^-20 for the exponential
(preactivations up to 16 of magnitude that count), four half units of FP32, and the preactivations' errors times
|act'| <= 1.2 and |act|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_amd as rr
from block_helpers import ACTIVATIONS, CODES, LEAST, ROUNDING, TYPES, Buf, assert_within, context
from mxfp4_cases import FORMS, TILE_SIZES, TILES
from test_gpu_block_offsets import OFFSETS, bounds

pytestmark = pytest.mark.gpu
ELEMENTS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


class Rows:
    """Random 4-bit rows on the GPU: packed elements, scale bytes [rows, blocks]."""

    def __init__(self, gen, rows, hidden, low, high):
        blocks = -(-hidden // 32)
        self.hidden = hidden
        self.q = torch.randint(0, 256, (rows, 16 * blocks), generator=gen, device="cuda:0", dtype=torch.uint8)
        if hidden % 32:  # (elements past the row's end are zeros)
            if hidden % 2:
                self.q[:, hidden // 2] &= 15
            self.q[:, (hidden + 1) // 2:] = 0
        self.scale = torch.randint(low, high + 1, (rows, blocks), generator=gen, device="cuda:0", dtype=torch.uint8)

    def values(self, at):
        """What rows `at` stand for."""
        q, scale = self.q[at], self.scale[at].double()
        table = torch.cat([ELEMENTS, -ELEMENTS]).to("cuda:0")
        v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], -1).reshape(*scale.shape, 32)
        power = torch.where(scale == 255, torch.full_like(scale, float("nan")), torch.exp2(scale - 127))
        return (v * power[..., None]).reshape(len(q), -1)

    def layout(self, pads):
        """The scales as the operators take them, `pads` in the bytes past a row's last block."""
        rows, blocks = self.scale.shape
        out = torch.full((rows, -(-blocks // 8) * 8), pads, dtype=torch.uint8, device="cuda:0")
        out[:, :blocks] = self.scale
        return out.view(rows, -1, 8).transpose(0, 1).contiguous()


def multiply(x, parts, offsets, n, dtype, act="silu", pads=255, stream=None):
    """y of rows x and one or two weights of experts * n channels."""
    rows, experts = len(x.q), len(offsets) - 1
    offs = Buf(torch.tensor(offsets, dtype=torch.int32, device="cuda:0"))
    operands = [[Buf(a.q), Buf(a.layout(pads))] for a in (x, *parts)]
    y = Buf(shape=(rows, n), dtype=TYPES[dtype], offset=1)
    up = dict(w_up=operands[2][0].ptr, w_up_scale=operands[2][1].ptr) if len(parts) == 2 else {}
    args = rr.Mxfp4GroupedGemmArgs(
        q=operands[0][0].ptr, q_scale=operands[0][1].ptr, w=operands[1][0].ptr, w_scale=operands[1][1].ptr, offsets=offs.ptr,
        y=y.ptr, rows=rows, experts=experts, hidden=x.hidden, output=n, activation=int(ACTIVATIONS[act][0]), dtype=CODES[dtype],
        **up)
    ctx, ws = context(rr.get_mxfp4_grouped_gemm_workspace_size(args), stream)
    status = rr.mxfp4_grouped_gemm(args, ctx)
    assert status.ok(), status.message
    assert all(buf.intact() for pair in operands for buf in pair) and offs.intact() and y.intact() and ws.intact()
    return y.t


def check(y, x, parts, at, n, dtype, act="silu", columns=None):
    """Rows at[e] .. at[e + 1] - 1 of y are expert e's, in `columns` (all of them by default); the others were left alone."""
    u, least, f32 = ROUNDING[dtype], LEAST[dtype], ROUNDING["f32"]
    inside = torch.zeros(len(y), dtype=torch.bool, device="cuda:0")
    columns = torch.arange(n, device="cuda:0") if columns is None else columns
    for e in range(len(at) - 1):
        if at[e] == at[e + 1]:
            continue
        inside[at[e]:at[e + 1]] = True
        rows = x.values(slice(at[e], at[e + 1]))
        wv = [part.values(e * n + columns).t().contiguous() for part in parts]
        p = [rows @ w for w in wv]
        err = [x.hidden * f32 * (rows.abs() @ w.abs()) for w in wv]
        want, bound = p[0], err[0]
        if len(parts) == 2:
            a = ACTIVATIONS[act][1](p[0])
            want = a * p[1]
            bound = (want.abs() * (2.0 ** -20 + 4 * f32) + 1.2 * (err[0] + p[0].abs() * 4 * f32) * (p[1].abs() + err[1])
                     + (a.abs() + 1.2 * err[0]) * err[1])
        got = y[at[e]:at[e + 1]][:, columns]
        if dtype == "f16":
            # from 65520 on (65504 and half a step) a result rounds to infinity; what may lie on either side is left out
            assert (torch.isinf(got) & (torch.sign(got) == torch.sign(want)))[want.abs() - bound >= 65520.0].all()
            fits = want.abs() + bound < 65504.0
            got, want, bound = got[fits], want[fits], bound[fits]
        assert_within(got, want, bound * (1 + u) + u * want.abs() + least, f"y of expert {e}")
    assert (y[~inside].contiguous().view(torch.uint8) == 0xA5).all()


def case(counts, k, n, gated, seed):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(seed)
    # (sums of random signs: near the square root of their length)
    x = Rows(gen, sum(counts) + 2, k, 124, 129)
    parts = [Rows(gen, len(counts) * n, k, 119, 124) for _ in range(1 + gated)]
    return x, parts, np.concatenate([[0], np.cumsum(counts)]).tolist()


@pytest.mark.parametrize("dtype,gated,act", FORMS)
@pytest.mark.parametrize("index", range(len(TILES)), ids=lambda i: f"{len(TILES[i][0])}x{sum(TILES[i][0])}-{TILES[i][1]}-{TILES[i][2]}-{TILES[i][3]}")
def test_products(device, index, dtype, gated, act):
    counts, k, n, _ = TILES[index]
    x, parts, offsets = case(counts, k, n, gated, index)
    check(multiply(x, parts, offsets, n, dtype, act), x, parts, offsets, n, dtype, act)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tile", list(TILE_SIZES))
@pytest.mark.parametrize("name", list(OFFSETS))
def test_offsets_that_do_not_rise(device, name, tile, dtype):
    """Bounds are cut to [0, rows], one that falls counts as the largest before it, rows of none are left alone."""
    per, n = TILE_SIZES[tile]
    experts = len(OFFSETS[name]) - 1
    rows = per * experts
    offsets = [rows * o // 10 for o in OFFSETS[name]]
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(experts)
    x = Rows(gen, rows, 320, 124, 129)
    w = Rows(gen, experts * n, 320, 119, 124)
    check(multiply(x, [w], offsets, n, dtype), x, [w], bounds(offsets, rows), n, dtype)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tile", list(TILE_SIZES))
def test_scales_over_the_whole_range(device, tile, dtype, gated):
    """Scales far apart whose products are ordinary numbers, the least and the largest, and NaN,
    which stays in its row or channel."""
    per, n = TILE_SIZES[tile]
    k, experts = 320, 4
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(tile)
    x = Rows(gen, per * experts, k, 127, 127)
    parts = [Rows(gen, experts * n, k, 127, 127) for _ in range(1 + gated)]
    shift = torch.randint(-120, 121, (10,), generator=gen, device="cuda:0")
    x.scale[:] = (127 + shift).to(torch.uint8)  # (every block its own)
    for part in parts:
        part.scale[:] = (127 - shift).to(torch.uint8)
        part.scale[0] = 254  # 2^127 ...
    x.scale[0] = 0  # ... and 2^-127
    bad_rows = [2, per + 31, per * experts - 1]
    bad_channels = [7, n - 1, experts * n - 1]
    for row, channel, block in zip(bad_rows, bad_channels, (4, 0, 9)):
        x.scale[row, block] = 255
        parts[-1].scale[channel, 9 - block] = 255
    y = multiply(x, parts, [per * e for e in range(experts + 1)], n, dtype).double()
    for e in range(experts):
        seg = slice(per * e, per * (e + 1))
        bad = torch.zeros(per, n, dtype=torch.bool, device="cuda:0")
        for row, channel in zip(bad_rows, bad_channels):
            if row // per == e:
                bad[row % per] = True
            if channel // n == e:
                bad[:, channel % n] = True
        assert torch.isnan(y[seg][bad]).all()
        rows, wv = x.values(seg), [part.values(slice(e * n, (e + 1) * n)).t().contiguous() for part in parts]
        size = [rows.abs() @ w.abs() for w in wv]
        fits = ~bad & (sum(size) < 1e15)
        assert fits.sum() >= (per - 2) * (n - 4)
        if gated:
            assert torch.isfinite(y[seg][fits]).all()
            continue
        want = rows @ wv[0]
        # (a block's part below the normal numbers may count as zero)
        bound = k * ROUNDING["f32"] * size[0] + 10 * 2.0 ** -126
        bound = bound * (1 + ROUNDING[dtype]) + ROUNDING[dtype] * want.abs()
        assert ((y[seg] - want).abs() <= bound)[fits].all()


@pytest.mark.parametrize("tile", list(TILE_SIZES))
def test_neighbours_do_not_leak(device, tile):
    """The rows and channels next to a ragged tile do not enter it."""
    per, n = TILE_SIZES[tile]
    k, experts = 72, 4
    rows = per * experts
    offsets = [0, 5, 5 + per, 4 * per - 5, 4 * per - 5]
    gen = torch.Generator(device="cuda:0")
    x, w = Rows(gen, rows, k, 127, 127), Rows(gen, experts * n, k, 127, 127)
    for part in (x, w):
        part.q[:, :k // 2] = 0x22  # ones
    w.scale[n:2 * n] = 130
    w.scale[2 * n:] = 120
    y = multiply(x, [w], offsets, n, "f32")
    assert (y[:5] == k).all() and (y[5:5 + per] == 8 * k).all() and (y[5 + per:rows - 5] == k / 128).all()
    assert (y[rows - 5:].contiguous().view(torch.uint8) == 0xA5).all()


@pytest.mark.parametrize("index", [0, 4, 10, 14])
def test_captured_on_a_stream(device, index):
    """Replayed from a graph with new rows between the replays, each replay the eager call's bits."""
    counts, k, n, _ = TILES[index]
    x, parts, offsets = case(counts, k, n, True, index)
    operands = [[a.q.clone(), a.layout(0)] for a in (x, *parts)]
    offs = torch.tensor(offsets, dtype=torch.int32, device="cuda:0")
    y, eager = (torch.zeros(len(x.q), n, dtype=torch.bfloat16, device="cuda:0") for _ in range(2))

    def run(out, stream):
        status = rr.mxfp4_grouped_gemm(rr.Mxfp4GroupedGemmArgs(
            q=operands[0][0].data_ptr(), q_scale=operands[0][1].data_ptr(), w=operands[1][0].data_ptr(),
            w_scale=operands[1][1].data_ptr(), w_up=operands[2][0].data_ptr(), w_up_scale=operands[2][1].data_ptr(),
            offsets=offs.data_ptr(), y=out.data_ptr(), rows=len(x.q), experts=len(counts), hidden=k, output=n),
            rr.RuntimeContext(stream=stream.cuda_stream, architecture=int(rr.DeviceArchitecture.kGfx950)))
        assert status.ok(), status.message

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        run(y, torch.cuda.current_stream())
    for _ in range(3):
        operands[0][0].copy_(operands[0][0].roll(1, 0))
        graph.replay()
        run(eager, torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
