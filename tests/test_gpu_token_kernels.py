"""Every kernel of sort_tokens, combine_tokens, their gradients and the 4-bit quantisation at sizes of its own
(token_cases.py), and the gate's gradient where every expert of a token is another. Bounds as in test_gpu_tokens.py."""
from __future__ import annotations

import pytest
import torch

import raggedroute_amd as rr
import test_gpu_mxfp4
import test_gpu_tokens as base
from block_helpers import LEAST, ROUNDING, TYPES, Buf, assert_within
from token_cases import COMBINE, MAPS, PAIRS, QUANTIZE, SORT, width

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,x_dtype", PAIRS)
@pytest.mark.parametrize("tokens,top_k,experts,pieces,whole", SORT)
def test_sort(device, tokens, top_k, experts, pieces, whole, dtype, x_dtype):
    ids = base.routes(tokens, top_k, experts, tokens + pieces)
    x = (torch.randn(tokens, width(dtype, pieces, whole), device="cuda:0") * 3).to(TYPES[x_dtype])
    for offset in (0, 1):
        base.check_sort(ids, x, experts, dtype, base.sort(ids, x, experts, dtype, x_dtype, offset))


@pytest.mark.parametrize("dtype,x_dtype", PAIRS)
@pytest.mark.parametrize("tokens,top_k,experts", MAPS)
def test_maps(device, tokens, top_k, experts, dtype, x_dtype):
    ids = base.routes(tokens, top_k, experts, tokens)
    b = base.sort(ids, torch.zeros(tokens, 8, device="cuda:0", dtype=TYPES[x_dtype]), experts, dtype, x_dtype, rows=False)
    offsets, pos, route = base.maps(ids, experts)
    assert torch.equal(b["offsets"].t.cpu(), offsets) and torch.equal(b["pos"].t.cpu(), pos)
    assert torch.equal(b["route"].t.cpu(), route) and b["out"].untouched(slice(None))


@pytest.mark.parametrize("dtype,y_dtype", PAIRS)
@pytest.mark.parametrize("tokens,top_k,pieces,whole", COMBINE)
def test_combine(device, tokens, top_k, pieces, whole, dtype, y_dtype):
    size = (tokens, top_k, 7, width(dtype, pieces, whole), "any")
    base.test_combine(device, *size, dtype, y_dtype)
    base.test_combine_backward(device, *size, dtype, y_dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,hidden", QUANTIZE)
def test_quantize(device, rows, hidden, dtype):
    test_gpu_mxfp4.test_quantize(device, rows, hidden, dtype)


@pytest.mark.parametrize("tokens,experts,top_k", [(200, 64, 2), (77, 130, 8), (33, 1024, 64), (1000, 3, 3), (5, 33, 33)])
def test_gate_backward_of_different_experts(device, tokens, experts, top_k):
    """A route's gradient takes a difference's rounding, top_k of the sum and one of the last product, of the terms'
    magnitudes: top_k + 2 half units, and their products with each other below one more. (Where an expert stands in
    several routes up to top_k - 1 additions follow, which is what the wider bound of (2 top_k + 3) allows.)"""
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(experts)
    ids = torch.rand(tokens, experts, device="cuda:0", generator=gen).topk(top_k, 1).indices.int()
    w = torch.softmax(8 * torch.randn(tokens, top_k, device="cuda:0", generator=gen), 1)
    dw = torch.randn(tokens, top_k, device="cuda:0", generator=gen)
    b = [Buf(ids), Buf(w), Buf(dw), Buf(shape=(tokens, experts), dtype=torch.float32)]
    base.run(rr.topk_gate_backward, rr.TopKGateBackwardArgs(
        expert_ids=b[0].ptr, weights=b[1].ptr, dweights=b[2].ptr, dlogits=b[3].ptr, tokens=tokens, experts=experts, top_k=top_k))
    assert all(buf.intact() for buf in b)
    terms = w.double()[:, :, None] * w.double()[:, None, :] * (dw.double()[:, :, None] - dw.double()[:, None, :])
    want, size = (torch.zeros(tokens, experts, dtype=torch.float64, device="cuda:0") for _ in range(2))
    want.scatter_(1, ids.long(), terms.sum(2))
    size.scatter_(1, ids.long(), terms.abs().sum(2))
    assert_within(b[3].t, want, (top_k + 3) * ROUNDING["f32"] * size + LEAST["f32"], "dlogits")
