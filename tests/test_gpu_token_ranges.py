"""The token and 4-bit operators at the ends of their ranges, the widest rows and outputs, and captured at sizes
whose calls are several launches."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_amd as rr
import test_gpu_mxfp4
import test_gpu_tokens as base
from block_helpers import CODES, TYPES, Buf
from test_gpu_mxfp4_tiles import Rows, multiply
from test_gpu_token_block import Calls, zeros

pytestmark = pytest.mark.gpu
MOST = 1 << 20  # columns


@pytest.mark.parametrize("dtype,x_dtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("tokens,top_k,experts", [(3, 3, 5), (70, 2, 9)])
@pytest.mark.parametrize("hidden", [MOST, MOST - 1])
def test_widest_rows(device, hidden, tokens, top_k, experts, dtype, x_dtype):
    ids = base.routes(tokens, top_k, experts, tokens)
    x = torch.randn(tokens, hidden, device="cuda:0").to(TYPES[x_dtype])
    base.check_sort(ids, x, experts, dtype, base.sort(ids, x, experts, dtype, x_dtype))
    if tokens == 3:
        base.test_combine(device, tokens, top_k, experts, hidden, "any", dtype, x_dtype)
        base.test_combine_backward(device, tokens, top_k, experts, hidden, "any", dtype, x_dtype)


@pytest.mark.parametrize("rows,hidden", [(2, MOST), (1, MOST - 1), (1030, 70001)])
def test_widest_rows_quantised(device, rows, hidden):
    test_gpu_mxfp4.test_quantize(device, rows, hidden, "bf16")


def ones(gen, rows, hidden):
    """Rows of 1 and -1: a sum of fewer than 2^24 of their products is exact in FP32, in any order."""
    out = Rows(gen, rows, hidden, 127, 127)
    bits = torch.randint(0, 4, out.q.shape, generator=gen, device="cuda:0", dtype=torch.uint8)
    out.q[:] = torch.tensor([0x22, 0x2A, 0xA2, 0xAA], dtype=torch.uint8, device="cuda:0")[bits.long()]
    if hidden % 32:
        if hidden % 2:
            out.q[:, hidden // 2] &= 15
        out.q[:, (hidden + 1) // 2:] = 0
    return out


# the kernel for few rows and both tile kernels: longest sums, then widest results
@pytest.mark.parametrize("counts,k,n", [([2, 1], MOST, 40), ([3], MOST - 1, 33), ([20] * 9, MOST, 513), ([300], MOST - 33, 2200),
                                        ([9, 11], 40, MOST), ([50], 64, MOST - 1), ([150], 33, MOST)])
def test_widest_products(device, counts, k, n):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(n)
    x, w = ones(gen, sum(counts), k), ones(gen, len(counts) * n, k)
    offsets = [sum(counts[:e]) for e in range(len(counts) + 1)]
    y = multiply(x, [w], offsets, n, "f32")
    columns = torch.cat([torch.arange(0, n, max(1, n // 100)), torch.arange(n - 33, n)]).cuda()
    for e in range(len(counts)):
        seg = slice(offsets[e], offsets[e + 1])
        want = x.values(seg) @ w.values(e * n + columns).t().contiguous()
        assert torch.equal(y[seg][:, columns].double(), want)


@pytest.mark.parametrize("tokens,top_k,experts,hidden", [(9000, 2, 7, 96), (3000, 8, 300, 257), (5000, 2, 5, 6000), (20, 2, 6, 100)])
def test_captured(device, tokens, top_k, experts, hidden):
    """Maps in one launch and two, rows in their own, sums, gradients and quantised rows, replayed from a graph with
    other routes and rows, eager work between the replays: the eager calls' bits each time."""
    rows, blocks = tokens * top_k, -(-hidden // 32)
    i32, f32, u8 = dict(dtype=torch.int32), dict(dtype=torch.float32), dict(dtype=torch.uint8)

    def step():
        t = dict(ids=zeros(tokens, top_k, **i32), x=zeros(tokens, hidden, **f32), dy=zeros(tokens, hidden, **f32),
                 weights=zeros(tokens, top_k, **f32), offsets=zeros(experts + 1, **i32), pos=zeros(rows, **i32),
                 route=zeros(rows, **i32), rows=zeros(rows, hidden), y=zeros(tokens, hidden, **f32), drows=zeros(rows, hidden),
                 dweights=zeros(tokens, top_k, **f32), dlogits=zeros(tokens, experts, **f32), dx=zeros(tokens, hidden, **f32),
                 q=zeros(rows, 16 * blocks, **u8), scale=zeros(-(-blocks // 8), rows, 8, **u8))
        p = {name: v.data_ptr() for name, v in t.items()}
        calls, bf16, fp32 = Calls(), CODES["bf16"], CODES["f32"]
        size = dict(tokens=tokens, top_k=top_k, hidden=hidden)
        calls.add("sort_tokens", rr.SortTokensArgs(x=p["x"], expert_ids=p["ids"], offsets=p["offsets"], route_pos=p["pos"],
                                                   sorted_route=p["route"], x_sorted=p["rows"], experts=experts, dtype=bf16,
                                                   x_dtype=fp32, **size))
        both = dict(y_sorted=p["rows"], route_pos=p["pos"], route_weights=p["weights"], dtype=bf16, y_dtype=fp32, **size)
        calls.add("combine_tokens", rr.CombineTokensArgs(y=p["y"], **both))
        calls.add("combine_tokens_backward", rr.CombineTokensBackwardArgs(dy=p["dy"], dy_sorted=p["drows"],
                                                                          droute_weights=p["dweights"], **both))
        calls.add("topk_gate_backward", rr.TopKGateBackwardArgs(expert_ids=p["ids"], weights=p["weights"], dweights=p["dweights"],
                                                                dlogits=p["dlogits"], tokens=tokens, experts=experts, top_k=top_k))
        calls.add("sort_tokens_backward", rr.SortTokensBackwardArgs(dx_sorted=p["drows"], route_pos=p["pos"], dx=p["dx"], dtype=bf16,
                                                                    x_dtype=fp32, **size))
        calls.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=p["x"], sorted_route=p["route"], q=p["q"], scale=p["scale"],
                                                                  rows=rows, dtype=fp32, **size))
        return t, calls

    (t, calls), (other, eager) = step(), step()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        calls.run(torch.cuda.current_stream())
    for seed in range(4):
        gen = torch.Generator(device="cuda:0")
        gen.manual_seed(seed)
        ids = torch.randint(-1, experts, (tokens, top_k), device="cuda:0", generator=gen, dtype=torch.int32)
        for name in ("x", "dy", "weights"):
            new = torch.randn(t[name].shape, device="cuda:0", generator=gen)
            t[name].copy_(new)
            other[name].copy_(new)
        t["ids"].copy_(ids)
        other["ids"].copy_(ids)
        # (rows behind the last one are left alone: of another replay's)
        for name in ("rows", "drows", "q", "scale"):
            t[name].zero_()
            other[name].zero_()
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        for name in t:
            assert torch.equal(t[name], other[name]), (seed, name)
    offsets, pos, route = base.maps(t["ids"].cpu(), experts)
    assert torch.equal(t["offsets"].cpu(), offsets) and torch.equal(t["pos"].cpu(), pos) and torch.equal(t["route"].cpu(), route)


# around the sizes from which another kernel ranks the routes, and numbers of experts from which others count them
@pytest.mark.parametrize("experts", [1, 2, 31, 32, 33, 255, 256, 257, 1023, 1024])
@pytest.mark.parametrize("tokens,top_k", [(127, 1), (64, 2), (43, 3), (8191, 1), (2731, 3), (16384, 1), (8192, 2), (2341, 7), (257, 64),
                                          (262144, 1), (131073, 2), (100001, 3), (4099, 64), (2 ** 20 + 1, 1)])
def test_maps_at_borders(device, tokens, top_k, experts):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(tokens + experts)
    routes = tokens * top_k
    for low, high in ((-1, experts + 1), (0, experts), (experts - 1, experts)):
        ids = torch.randint(low, high, (routes,), device="cuda:0", generator=gen, dtype=torch.int32)
        b = dict(ids=Buf(ids), offsets=Buf(shape=(experts + 1,), dtype=torch.int32), pos=Buf(shape=(routes,), dtype=torch.int32),
                 route=Buf(shape=(routes,), dtype=torch.int32))
        base.run(rr.sort_tokens, rr.SortTokensArgs(
            expert_ids=b["ids"].ptr, offsets=b["offsets"].ptr, route_pos=b["pos"].ptr, sorted_route=b["route"].ptr, tokens=tokens,
            experts=experts, top_k=top_k), rr.get_sort_tokens_workspace_size)
        assert all(buf.intact() for buf in b.values())
        key = torch.where((ids >= 0) & (ids < experts), ids, experts).long()
        counts = torch.bincount(key, minlength=experts + 1)[:experts]
        placed = int(counts.sum())
        order = torch.sort(key, stable=True).indices[:placed].int()
        offsets = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda:0"), counts.cumsum(0)]).int()
        pos = torch.full((routes,), -1, dtype=torch.int32, device="cuda:0")
        pos[order.long()] = torch.arange(placed, dtype=torch.int32, device="cuda:0")
        assert torch.equal(b["offsets"].t, offsets) and torch.equal(b["pos"].t, pos)
        assert torch.equal(b["route"].t[:placed], order) and (b["route"].t[placed:] == -1).all()


@pytest.mark.parametrize("dtype,least", [("f16", -24), ("bf16", -133), ("f32", -149)])
def test_quantised_subnormal_numbers(device, dtype, least):
    """Rows of multiples of the type's least number, alone and beside ordinary ones."""
    x = torch.zeros(40, 64, dtype=torch.float64)
    x[:, :32] = torch.arange(40 * 32, dtype=torch.float64).view(40, 32) % 67 - 33
    x = torch.ldexp(x, torch.tensor(least))
    x[20:, 40] = 1.5
    x = x.to(TYPES[dtype])
    assert x[:, :32].any(1).all()
    code, scale = test_gpu_mxfp4.encode(x.double().numpy())
    q, s = test_gpu_mxfp4.quantize(x.cuda(), dtype)
    assert np.array_equal(s, test_gpu_mxfp4.layout(scale))
    test_gpu_mxfp4.same_codes(q, test_gpu_mxfp4.pack(code))
