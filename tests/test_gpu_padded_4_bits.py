"""Two 4-bit products with a quantisation between them over a padded batch: rows behind the last segment are
quantised with whatever they hold, and nothing that a token gets depends on them."""
from __future__ import annotations

import pytest
import torch

import raggedroute_amd as rr
from block_helpers import CODES
from test_gpu_mxfp4_tiles import Rows
from test_gpu_token_block import Calls, zeros

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,top_k,experts,hidden,inner", [(9, 2, 8, 320, 130), (1500, 2, 6, 100, 1200), (700, 4, 300, 64, 70)])
def test_rows_behind_the_last_segment(device, tokens, top_k, experts, hidden, inner):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(tokens)
    rows = tokens * top_k
    x = torch.randn(tokens, hidden, device="cuda:0", generator=gen).bfloat16()
    w = torch.rand(tokens, top_k, device="cuda:0", generator=gen)
    ids = torch.randint(0, experts, (tokens, top_k), device="cuda:0", generator=gen, dtype=torch.int32)
    ids[tokens // 3:tokens // 2] = -1  # padding tokens, and single routes of others
    ids[-1, 0] = experts
    weights = [Rows(gen, experts * inner, hidden, 119, 122), Rows(gen, experts * inner, hidden, 119, 122), Rows(gen, experts * hidden, inner, 119, 122)]
    scales = [part.layout(255) for part in weights]
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        u8, i32 = dict(dtype=torch.uint8), dict(dtype=torch.int32)
        t = dict(offsets=zeros(experts + 1, **i32), pos=zeros(rows, **i32), route=zeros(rows, **i32))
        for name, k in (("x", hidden), ("a", inner)):
            blocks = -(-k // 32)
            t["q" + name], t["s" + name] = zeros(rows, 16 * blocks, **u8), zeros(-(-blocks // 8), rows, 8, **u8)
        t |= dict(a=torch.full((rows, inner), fill, dtype=torch.bfloat16, device="cuda:0"),
                  r=torch.full((rows, hidden), fill, dtype=torch.bfloat16, device="cuda:0"), y=zeros(tokens, hidden))
        p = {name: v.data_ptr() for name, v in t.items()}
        calls = Calls()
        calls.add("sort_tokens", rr.SortTokensArgs(expert_ids=ids.data_ptr(), offsets=p["offsets"], route_pos=p["pos"],
                                                   sorted_route=p["route"], tokens=tokens, experts=experts, top_k=top_k))
        calls.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=x.data_ptr(), sorted_route=p["route"], q=p["qx"], scale=p["sx"],
                                                                  rows=rows, hidden=hidden, tokens=tokens, top_k=top_k))
        common = dict(offsets=p["offsets"], rows=rows, experts=experts)
        calls.add("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
            q=p["qx"], q_scale=p["sx"], w=weights[0].q.data_ptr(), w_scale=scales[0].data_ptr(), w_up=weights[1].q.data_ptr(),
            w_up_scale=scales[1].data_ptr(), y=p["a"], hidden=hidden, output=inner, **common))
        calls.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=p["a"], q=p["qa"], scale=p["sa"], rows=rows, hidden=inner))
        calls.add("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
            q=p["qa"], q_scale=p["sa"], w=weights[2].q.data_ptr(), w_scale=scales[2].data_ptr(), y=p["r"], hidden=inner,
            output=hidden, **common))
        calls.add("combine_tokens", rr.CombineTokensArgs(y_sorted=p["r"], route_pos=p["pos"], route_weights=w.data_ptr(), y=p["y"],
                                                         tokens=tokens, top_k=top_k, hidden=hidden, dtype=CODES["bf16"]))
        calls.run()
        torch.cuda.synchronize()
        placed = int(t["offsets"][-1])
        assert placed == int(((ids >= 0) & (ids < experts)).sum()) < rows
        for name in ("a", "r"):  # (left alone)
            behind = t[name][placed:]
            assert torch.equal(torch.nan_to_num(behind, nan=1.0), torch.nan_to_num(torch.full_like(behind, fill), nan=1.0))
        bad = t["sa"].transpose(0, 1).reshape(rows, -1)[:, :-(-inner // 32)] == 255
        assert not bad[:placed].any() and bool(bad[placed:].all()) == (fill != 0.0)
        results.append(t["y"])
    assert torch.isfinite(results[0]).all() and results[0].any() and not results[0][tokens // 3:tokens // 2].any()
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])
