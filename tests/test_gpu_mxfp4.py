"""quantize_rows_mxfp4 and mxfp4_grouped_gemm against their definitions.

Quantisation is exact (powers of two, a rounding to even). A product's terms are exact; their sum
over n elements takes at most n roundings to FP32 of partial sums no larger than the sum of the
terms' magnitudes, and the result is rounded to its type; the gated form adds 2^-20 for the
exponential, four half units of FP32, and the preactivation's error times |act'| <= 1.2.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_amd as rr
from block_helpers import ACTIVATIONS, CODES, LEAST, ROUNDING, TYPES, Buf, assert_within, context, offsets_of, segments

pytestmark = pytest.mark.gpu
FAMILIES = {"auto": rr.kernel(), "naive": rr.kernel(rr.KernelFamily.kNaive)}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(x):
    """float64 rows [rows, hidden] to (codes [rows, 32 blocks], scale bytes [rows, blocks])."""
    rows, hidden = x.shape
    v = np.zeros((rows, -(-hidden // 32) * 32))
    v[:, :hidden] = x
    v = v.reshape(rows, -1, 32)
    top = np.abs(v).max(2)
    finite = np.isfinite(top)
    power = np.frexp(np.where(finite & (top > 0), top, 1.0))[1] - 1 - 2
    power = np.where(finite & (top > 0), np.maximum(power, -127), -127)
    a = np.abs(np.where(finite[:, :, None], v, 0.0)) / np.exp2(power)[:, :, None]
    code = np.zeros(v.shape, dtype=np.uint8)
    for c in range(7):
        middle = (E2M1[c] + E2M1[c + 1]) / 2
        code += (a > middle if c % 2 == 0 else a >= middle).astype(np.uint8)
    code |= np.where(np.signbit(v) & (code > 0), 8, 0).astype(np.uint8)
    code[~finite] = 0
    return code.reshape(rows, -1), np.where(finite, power + 127, 255).astype(np.uint8)


def pack(code):
    return code[:, 0::2] | code[:, 1::2] << 4


def layout(scale):
    """Scale bytes [rows, blocks] in the operators' order [slices, rows, 8]."""
    rows, blocks = scale.shape
    out = np.zeros((rows, -(-blocks // 8) * 8), dtype=np.uint8)
    out[:, :blocks] = scale
    return np.ascontiguousarray(out.reshape(rows, -1, 8).transpose(1, 0, 2))


def values(code, scale):
    v = np.concatenate([E2M1, -E2M1])[code].reshape(*scale.shape, 32)
    power = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return (v * power[..., None]).reshape(code.shape)


def quantize(x, dtype, offset=0, route=None, rows=None, top_k=2):
    tokens, hidden = x.shape
    rows = tokens if rows is None else rows
    blocks, slices = -(-hidden // 32), -(-hidden // 256)
    q, s = Buf(shape=(rows, 16 * blocks), dtype=torch.uint8), Buf(shape=(slices, rows, 8), dtype=torch.uint8)
    xb = Buf(x, offset=offset)
    rb = Buf(route, offset=offset) if route is not None else None
    ctx, _ = context()
    status = rr.quantize_rows_mxfp4(rr.QuantizeRowsMxfp4Args(
        x=xb.ptr, sorted_route=rb.ptr if rb else None, q=q.ptr, scale=s.ptr, rows=rows, hidden=hidden, tokens=tokens,
        top_k=top_k, dtype=CODES[dtype]), ctx)
    assert status.ok(), status.message
    assert q.intact() and s.intact() and xb.intact()
    return q.t.cpu().numpy(), s.t.cpu().numpy()


def same_codes(got, want):
    """Packed elements equal, whichever sign a zero has."""
    for shift in (0, 4):
        g, w = got >> shift & 15, want >> shift & 15
        assert np.array_equal(np.where(g == 8, 0, g), np.where(w == 8, 0, w))


@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (2, 32), (5, 33), (4, 255), (3, 256), (2, 257), (7, 500), (3, 1023),
                                         (2, 1024), (9, 2049), (300, 96), (2, 8190), (1, 20001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantize(device, rows, hidden, dtype):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(rows * hidden)
    x = torch.randn(rows, hidden, device="cuda:0", generator=gen)
    x *= torch.exp2(torch.randint(-12, 12, (rows, hidden), device="cuda:0", generator=gen).float() * 0.25)
    if rows > 2:
        x[0] = 0.0
    x = x.to(TYPES[dtype])
    code, scale = encode(x.double().cpu().numpy())
    for offset in (0, 1):
        q, s = quantize(x, dtype, offset)
        assert np.array_equal(s, layout(scale))
        same_codes(q, pack(code))


def test_quantize_borders(device):
    """Every border between two elements, its neighbours in FP32, at scales over the whole range,
    the largest and the subnormal numbers."""
    middles = (E2M1[:-1] + E2M1[1:]) / 2
    points = np.concatenate([E2M1, middles, [7.0, 7.999999]]).astype(np.float32)
    points = np.concatenate([points, np.nextafter(points, np.float32(8)), np.nextafter(points, np.float32(-8))])
    rows = []
    for power in (-149, -140, -130, -127, -126, -125, -100, -1, 0, 1, 60, 120, 124, 125):
        with np.errstate(over="ignore"):
            v = np.ldexp(points.astype(np.float64), power)
            v = v[np.abs(v) <= np.finfo(np.float32).max].astype(np.float32)
        for i in range(0, len(v), 31):
            row = np.zeros(32, dtype=np.float32)
            row[:len(v[i:i + 31])] = v[i:i + 31]
            row[31] = np.float32(np.ldexp(4.0, min(power, 125)))  # the block's power is the one meant
            rows.append(row * np.where(np.arange(32) % 3 == 0, -1, 1).astype(np.float32))
    x = np.stack(rows)
    code, scale = encode(x.astype(np.float64))
    q, s = quantize(torch.from_numpy(x).cuda(), "f32")
    assert np.array_equal(s, layout(scale))
    same_codes(q, pack(code))


def test_quantize_special_values(device):
    x = torch.ones(4, 96, device="cuda:0")
    x[1, 3], x[2, 40], x[3, 95] = float("inf"), float("nan"), float("-inf")
    q, s = quantize(x, "f32")
    bad = np.zeros((4, 3), dtype=bool)
    bad[1, 0] = bad[2, 1] = bad[3, 2] = True
    assert np.array_equal(s[0, :, :3] == 255, bad) and (s[0, :, 3:] == 0).all()
    elements = q.reshape(4, 3, 16)
    assert (elements[bad] == 0).all() and (elements[~bad] == 0x66).all()  # 1 = 4 * 2^-2


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_gathered(device, dtype):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(3)
    x = torch.randn(20, 300, device="cuda:0", generator=gen).to(TYPES[dtype])
    route = torch.tensor([59, 0, 1, 2, 30, 30, -1, 60, 2 ** 31 - 1, -2 ** 31, 7], dtype=torch.int32, device="cuda:0")
    q, s = quantize(x, dtype, 1, route, rows=11, top_k=3)
    code, scale = encode(x.double().cpu().numpy())
    r = route.cpu().numpy()
    good = (r >= 0) & (r < 60)
    same_codes(q[good], pack(code)[r[good] // 3])
    assert np.array_equal(s[:, good], layout(scale)[:, r[good] // 3])
    assert (q[~good] == 0xA5).all() and (s[:, ~good] == 0xA5).all()


def weights(gen, rows, hidden, spread=3):
    """Random elements and scales: (packed, scale bytes [rows, blocks], values)."""
    blocks = -(-hidden // 32)
    code = gen.integers(0, 16, (rows, 32 * blocks), dtype=np.uint8)
    code[:, hidden:] = 0
    scale = gen.integers(127 - spread, 128 + spread, (rows, blocks), dtype=np.uint8)
    return pack(code), scale, values(code, scale)


def product(q, q_scale, w, w_scale, counts, hidden, n, dtype, act, family, pads=0):
    rows = q.shape[0]
    e = len(counts)

    def scales(s):
        out = layout(s)
        if s.shape[1] % 8 and pads:
            out[-1, :, s.shape[1] % 8:] = pads
        return Buf(torch.from_numpy(out).cuda())

    dev = lambda a: Buf(torch.from_numpy(np.ascontiguousarray(a)).cuda())  # noqa: E731
    bufs = [dev(q), scales(q_scale), *(dev(a) for a in w), *(scales(s) for s in w_scale)]
    gated = len(w) == 2
    offs = Buf(offsets_of(counts)[0])
    y = Buf(shape=(rows, n), dtype=TYPES[dtype], offset=1)
    args = rr.Mxfp4GroupedGemmArgs(
        q=bufs[0].ptr, q_scale=bufs[1].ptr, w=bufs[2].ptr, w_scale=bufs[2 + len(w)].ptr,
        w_up=bufs[3].ptr if gated else None, w_up_scale=bufs[5].ptr if gated else None, offsets=offs.ptr, y=y.ptr,
        rows=rows, experts=e, hidden=hidden, output=n, activation=int(ACTIVATIONS[act][0]), dtype=CODES[dtype],
        kernel=FAMILIES[family])
    ctx, ws = context(rr.get_mxfp4_grouped_gemm_workspace_size(args))
    status = rr.mxfp4_grouped_gemm(args, ctx)
    assert status.ok(), status.message
    for buf in (*bufs, offs, y, ws):
        assert buf.intact()
    return y


SHAPES = [
    ([1], 1, 1),
    ([2, 0, 1], 16, 3),
    ([0, 5, 0, 17, 1, 0], 33, 47),
    ([16, 15], 64, 64),
    ([0, 3], 256, 128),
    ([1, 1, 0, 6], 520, 272),
    ([70, 0, 31], 144, 200),
    ([129, 64, 1], 257, 130),
    ([256, 300], 768, 264),
    ([600, 9], 1040, 512),
    ([0, 37, 0, 1, 2] + [0] * 9, 2080, 96),
    ([513], 1000, 700),
    ([40] * 7 + [0, 130], 300, 33),
]


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("dtype,gated,act", [("f32", False, "silu"), ("bf16", True, "silu"), ("f16", True, "gelu"),
                                             ("bf16", False, "silu"), ("f32", True, "silu"), ("f16", False, "silu")])
@pytest.mark.parametrize("counts,k,n", SHAPES)
def test_products(device, counts, k, n, dtype, gated, act, family):
    gen = np.random.default_rng(k * n)
    rows, e = sum(counts) + 2, len(counts)
    q, qs, qv = weights(gen, rows, k)
    parts = [weights(gen, e * n, k) for _ in range(1 + gated)]
    # (sums of random signs: near the square root of their length)
    parts = [(p, s - 5, v / 32) for p, s, v in parts]
    y = product(q, qs, [p[0] for p in parts], [p[1] for p in parts], counts, k, n, dtype, act, family, pads=255).t
    u, least, f32 = ROUNDING[dtype], LEAST[dtype], ROUNDING["f32"]
    qv = torch.from_numpy(qv).cuda()
    for x, seg in segments(counts):
        wv = [torch.from_numpy(p[2]).cuda().view(e, n, -1)[x].t().contiguous() for p in parts]
        p = [qv[seg] @ w for w in wv]
        err = [k * f32 * (qv[seg].abs() @ w.abs()) for w in wv]
        if gated:
            a = ACTIVATIONS[act][1](p[0])
            want = a * p[1]
            bound = (want.abs() * (2.0 ** -20 + 4 * f32) + 1.2 * (err[0] + p[0].abs() * 4 * f32) * (p[1].abs() + err[1])
                     + (a.abs() + 1.2 * err[0]) * err[1])
        else:
            want, bound = p[0], err[0]
        got = y[seg]
        if dtype == "f16":
            # from 65520 on (65504 and half a step) a result rounds to infinity; what may lie on either side is left out
            assert (torch.isinf(got) & (torch.sign(got) == torch.sign(want)))[want.abs() - bound >= 65520.0].all()
            inside = want.abs() + bound < 65504.0
            got, want, bound = got[inside], want[inside], bound[inside]
        assert_within(got, want, bound * (1 + u) + u * want.abs() + least, f"y of expert {x}")
    assert (y[sum(counts):].contiguous().view(torch.uint8) == 0xA5).all()


# Sums of many slices by two, four and eight waves, with few workgroups (half the columns each) and with more.
SHARED = [
    ([1], 4097, 1),
    ([1, 1, 0, 6], 4129, 272),
    ([0, 17, 0], 14337, 63),
    ([3, 33], 2049, 250),
    ([20, 3], 1100, 97),
    ([20, 3], 2050, 5501),
    ([20, 3], 4100, 5501),
    ([2, 0, 1], 4100, 4160),
    ([20, 3], 800, 5501),
]


@pytest.mark.parametrize("dtype,gated,act", [("bf16", False, "silu"), ("f32", True, "gelu")])
@pytest.mark.parametrize("counts,k,n", SHARED)
def test_products_of_shared_sums(device, counts, k, n, dtype, gated, act):
    test_products(device, counts, k, n, dtype, gated, act, "auto")


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("rows", [5, 300])
def test_scales_over_the_whole_range(device, rows, family):
    """Scales far apart whose products are ordinary numbers, the least and the largest, and NaN,
    which stays in its row or channel."""
    k, n = 320, 48
    gen = np.random.default_rng(rows)
    q, qs, _ = weights(gen, rows, k)
    w, ws, _ = weights(gen, n, k)
    shift = gen.integers(-120, 121, 10)
    qs[:], ws[:] = 127 + shift, 127 - shift  # (every block its own)
    qs[2, 4] = 255
    ws[7, 9] = 255
    qs[0], ws[0] = 0, 254  # 2^-127 and 2^127
    wide = [values(np.stack([p & 15, p >> 4], -1).reshape(len(p), -1), s) for p, s in ((q, qs), (w, ws))]
    y = product(q, qs, [w], [ws], [rows], k, n, "f32", "silu", family).t.cpu().double().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        want = wide[0] @ wide[1].T
        size = np.abs(wide[0]) @ np.abs(wide[1]).T
    bad = np.zeros_like(want, dtype=bool)
    bad[2], bad[:, 7] = True, True
    assert np.isnan(y[bad]).all()
    fits = ~bad & (size < 1e38)
    assert fits.sum() > fits.size // 2
    assert (np.abs(y - want)[fits] <= k * 2.0 ** -24 * size[fits] + 2.0 ** -126).all()


def test_neighbours_do_not_leak(device):
    """The rows and channels next to a ragged tile do not enter it."""
    counts, k, n = [5, 130, 290], 72, 72
    rows = sum(counts) + 5
    q = np.full((rows, 48), 0x22, dtype=np.uint8)
    q[:, 36:] = 0
    qs = np.full((rows, 3), 127, dtype=np.uint8)
    w = np.full((3 * n, 48), 0x22, dtype=np.uint8)
    w[:, 36:] = 0
    ws = np.full((3 * n, 3), 127, dtype=np.uint8)
    ws[n:2 * n] = 130
    ws[2 * n:] = 120
    y = product(q, qs, [w], [ws], counts, k, n, "f32", "silu", "auto").t
    assert (y[:5] == k).all() and (y[5:135] == 8 * k).all() and (y[135:425] == k / 128).all()


def test_quantised_rows_multiplied(device):
    """Both operators in a row, rows gathered: 4-bit rows of an identity's products."""
    k, tokens, top_k = 96, 30, 2
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(1)
    x = torch.randn(tokens, k, device="cuda:0", generator=gen)
    route = torch.randperm(tokens * top_k, device="cuda:0", generator=gen).int()
    q, s = quantize(x, "f32", 0, route, rows=60)
    eye, eye_scale = encode(np.eye(k))
    y = Buf(shape=(60, k), dtype=torch.float32)
    dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (q, s, pack(eye), layout(eye_scale))]
    offs = torch.tensor([0, 60], dtype=torch.int32, device="cuda:0")
    ctx, _ = context()
    status = rr.mxfp4_grouped_gemm(rr.Mxfp4GroupedGemmArgs(
        q=dev[0].data_ptr(), q_scale=dev[1].data_ptr(), w=dev[2].data_ptr(), w_scale=dev[3].data_ptr(),
        offsets=offs.data_ptr(), y=y.ptr, rows=60, experts=1, hidden=k, output=k, dtype=CODES["f32"]), ctx)
    assert status.ok(), status.message
    code, scale = encode(x.double().cpu().numpy())
    want = values(code, scale)[route.cpu().numpy() // top_k]
    assert np.array_equal(y.t.cpu().double().numpy(), want)
