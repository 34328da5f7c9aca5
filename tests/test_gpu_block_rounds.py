"""The expert block's kernels over more work than workgroups: whole and partial rounds of tiles,
full and short tiles one after the other, slices that run on into the next tile, and rows of
the norms and of the quantisation that one workgroup takes in turn. Value by value against 64
bits, with the bounds of the other tests, and twice for equal bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from block_helpers import ACTIVATIONS, LEAST, ROUNDING, TYPES, assert_within, offsets_of, segments
from test_gpu_block_ffn import backward, check_backward, check_forward, forward, make
from test_gpu_block_int8 import product, quantize
from test_gpu_block_norm import backward as norm_backward
from test_gpu_block_norm import check_backward as check_norm_backward
from test_gpu_block_norm import check_forward as check_norm_forward
from test_gpu_block_norm import forward as norm_forward
from test_gpu_block_norm import make as make_norm

pytestmark = pytest.mark.gpu

# eight experts of long segments: 24 row tiles of 256 (five of them short), 43 of 128
LONG = [1000, 300, 0, 513, 2049, 129, 257, 640]
# seventy of short ones, on both sides of a slice, half a tile and a tile of 128 rows: 91 tiles
SHORT = [0, 1, 63, 64, 65, 127, 128, 129, 200, 300] * 7


def same_bits(first, again):
    for name in first:
        assert torch.equal(first[name].raw, again[name].raw), name


FFN = [
    # tiles of 256 rows: 528 (gate and up, paired weight gradients), 264 (gradients of gate and up, of Wd)
    (LONG, 600, 2816, 600, "bf16", "silu"),
    # 264 (down, data gradients): one round and eight tiles, cut into four
    (LONG, 2816, 136, 2816, "f16", "gelu"),
    # one slice a tile, and none in two experts of three
    (LONG + [0] * 7, 64, 2816, 1032, "bf16", "gelu"),
    # 256 tiles: one round, nothing left
    ([4096], 72, 2048, 4096, "f16", "silu"),
    # tiles of 128 rows, three stages: 364 (gate and up), 560 (gradients of Wd); 364 (down), 273 (data
    # gradients); 364 (gradients of gate and up)
    (SHORT, 136, 512, 264, "bf16", "silu"),
    (SHORT, 520, 264, 776, "f16", "silu"),
    (SHORT, 72, 776, 72, "bf16", "gelu"),
    # through registers: 516, 86 and 258 tiles
    (LONG, 333, 1501, 601, "bf16", "silu"),
    (LONG, 1501, 333, 1501, "f16", "gelu"),
    (SHORT, 77, 515, 333, "bf16", "gelu"),
]


@pytest.mark.parametrize("counts,k,f,n,dtype,act", FFN)
def test_ffn_forward(device, counts, k, f, n, dtype, act):
    v, b, rows = make(counts, k, f, n, dtype, seed=k + f)
    out = forward(b, counts, rows, k, f, n, dtype, act)
    check_forward(v, out, counts, dtype, act)
    same_bits(out, forward(b, counts, rows, k, f, n, dtype, act))


@pytest.mark.parametrize("counts,k,f,n,dtype,act", FFN)
def test_ffn_backward(device, counts, k, f, n, dtype, act):
    v, b, rows = make(counts, k, f, n, dtype, seed=f + n)
    out = backward(b, counts, rows, k, f, n, dtype, act)
    check_backward(v, out, counts, dtype, act)
    same_bits(out, backward(b, counts, rows, k, f, n, dtype, act))


@pytest.mark.parametrize("k,f,n", [(264, 136, 200), (77, 65, 131)])
@pytest.mark.parametrize("experts", [16, 128])
def test_all_rows_on_one_expert(device, experts, k, f, n):
    """At the most rows that the kernel for few rows an expert takes, five on average."""
    counts = [0] * (experts // 3) + [5 * experts] + [0] * (experts - experts // 3 - 1)
    v, b, rows = make(counts, k, f, n, "bf16", seed=experts)
    check_forward(v, forward(b, counts, rows, k, f, n, "bf16"), counts, "bf16", "silu")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts,k,n,dtype", [(LONG, 208, 2816, "bf16"), (LONG, 128, 2816, "f32"), ([4096], 144, 4096, "f16"),
                                              ([c // 2 for c in SHORT], 272, 1040, "f32"), (LONG, 77, 1501, "bf16"),
                                              ([0] * 42 + [384] + [0] * 85, 272, 200, "f32")])
def test_int8(device, counts, k, n, dtype, gated):
    """Bounds as for single tiles: four half units of FP32 and one of the type; the gated form's
    exponential 2^-20, and the preactivation's error 1.2 times."""
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(k + n)
    _, rows = offsets_of(counts)
    e = len(counts)
    q = torch.randint(-127, 128, (rows, k), device="cuda:0", generator=gen, dtype=torch.int8)
    qs = torch.rand(rows, device="cuda:0", generator=gen) * 0.02 + 0.001
    weights = [torch.randint(-127, 128, (e, n, k), device="cuda:0", generator=gen, dtype=torch.int8)
               for _ in range(1 + gated)]
    scales = [(torch.rand(e, n, device="cuda:0", generator=gen) + 0.1) * 0.02 * k ** -0.5 for _ in weights]
    y = product(q, qs, weights, scales, counts, n, dtype, "silu", "auto")
    u, least, f32 = ROUNDING[dtype], LEAST[dtype], 4 * ROUNDING["f32"]
    got = y.t
    for x, seg in segments(counts):
        p = [(q[seg].double() @ w[x].double().t().contiguous()) * qs[seg, None].double() * s[x].double()
             for w, s in zip(weights, scales)]
        if gated:
            want = ACTIVATIONS["silu"][1](p[0]) * p[1]
            bound = (want.abs() * (2.0 ** -20 + f32) + 1.2 * p[0].abs() * f32 * p[1].abs()) * (1 + u) + u * want.abs()
        else:
            want = p[0]
            bound = want.abs() * (u + f32 * (1 + u))
        assert_within(got[seg], want, bound + least, f"y of expert {x}")
    same_bits({"y": y}, {"y": product(q, qs, weights, scales, counts, n, dtype, "silu", "auto")})


# rows past the workgroups of a launch: 262144 threads' worth
@pytest.mark.parametrize("t,d,gate_tokens,dtype,block_dtype",
                         [(9001, 96, 50, "bf16", "bf16"), (9001, 520, 1, "f16", "f32"), (2501, 4096, 7, "bf16", "f32"),
                          (1100, 8191, 0, "bf16", "bf16"), (701, 16384, 3, "f16", "f16"), (701, 8192, 300, "f32", "f32"),
                          (601, 17001, 4, "bf16", "bf16"), (601, 9001, 0, "f32", "f32")])
def test_norm_forward(device, t, d, gate_tokens, dtype, block_dtype):
    v = make_norm(t, d, dtype, block_dtype, gate_tokens, seed=t + d)
    got = norm_forward(v, t, d, dtype, block_dtype, gate_tokens)
    check_norm_forward(v, got, dtype, gate_tokens)
    again = norm_forward(v, t, d, dtype, block_dtype, gate_tokens)
    assert all(torch.equal(got[name], again[name]) for name in got)


# parts of about five tokens, with gate rows of one, of a few, of more than a part, and none
@pytest.mark.parametrize("t,d,dtype,block_dtype", [(1300, 8192, "bf16", "bf16"), (701, 16384, "bf16", "bf16"),
                                                   (701, 16001, "f16", "f32"), (701, 8192, "f32", "f32"),
                                                   (601, 17001, "bf16", "f32"), (601, 9001, "f32", "f32")])
@pytest.mark.parametrize("gate_tokens", [0, 1, 2, 4, 300])
def test_norm_backward(device, t, d, gate_tokens, dtype, block_dtype):
    v = make_norm(t, d, dtype, block_dtype, gate_tokens, seed=t + d + gate_tokens)
    v["h"] = v.pop("x")
    got = norm_backward(v, t, d, dtype, block_dtype, gate_tokens)
    check_norm_backward(v, got, dtype, block_dtype, gate_tokens)
    again = norm_backward(v, t, d, dtype, block_dtype, gate_tokens)
    assert all(torch.equal(got[name], again[name]) for name in got)


@pytest.mark.parametrize("rows,hidden,dtype", [(9001, 264, "bf16"), (5000, 900, "f32"), (2501, 4096, "f16"),
                                               (701, 16384, "bf16"), (701, 8192, "f32"), (601, 17001, "bf16")])
def test_quantize_rows(device, rows, hidden, dtype):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(rows + hidden)
    x = torch.randn(rows, hidden, device="cuda:0", generator=gen)
    x *= torch.logspace(-3, 3, rows, device="cuda:0")[:, None]
    x = x.to(TYPES[dtype])
    q, s = quantize(x, dtype)
    host = x.float().cpu().numpy()
    scale = (np.abs(host).max(axis=1) / np.float32(127.0)).astype(np.float32)
    assert np.array_equal(s.t.cpu().numpy(), scale)
    assert np.array_equal(q.t.cpu().numpy(), np.rint(host / scale[:, None]).astype(np.int8))
