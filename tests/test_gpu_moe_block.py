"""The expert block's operators together with the routing chain (examples/moe_block.py),
against the same block in 64-bit torch."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "moe_block.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_block_example", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def norm(v, w, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w


def plain(block, x, ids, weights, p):
    """h and the next input in 64 bits, with the routes given."""
    n = norm(x, p["pre"], block.eps)
    y = torch.zeros_like(x)
    for e in range(block.experts):
        token, rank = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            a = torch.nn.functional.silu(n[token] @ p["w_gate"][e]) * (n[token] @ p["w_up"][e])
            y = y.index_add(0, token, weights[token, rank][:, None] * (a @ p["w_down"][e]))
    h = x + block.scale * norm(y, p["post"], block.eps)
    return h, norm(h, p["next"], block.eps)


def relative(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("tokens,hidden,inner,experts", [(1, 64, 32, 4), (37, 96, 72, 8), (200, 128, 64, 40),
                                                         (300, 60, 33, 5)])
def test_block(device, example, tokens, hidden, inner, experts):
    """Forward: the rows' rounding to BF16 enters g and u (2^-9 of a value each, up to 1.5
    times as much through the activation) and a's once more, at most 5 * 2^-9 in norm, which
    the norm after the block keeps: 2^-6. Backward: the same again for the gradients' rows,
    dg and du, the kept g, u and a and the result: 2^-5. Int8: half a step of max / 127 on
    rows, weights and a, whose largest value is up to eight times its root mean square:
    2^-3."""
    block = example.MoeBlock(hidden, inner, experts, seed=tokens)
    block.quantize()
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(7 * tokens)
    x, dh, dn = (torch.randn(tokens, hidden, device="cuda:0", generator=gen) for _ in range(3))
    h, n, kept = block.forward(x, keep=True)
    grads = block.backward(kept, dh, dn)
    served, _ = block.forward_int8(x)

    ids, weights = kept["routes"]["ids"].cpu().long(), kept["routes"]["weights"].double().cpu()
    logits = norm(x.double(), block.pre.double(), block.eps) @ block.router.double()
    logits = logits.cpu()  # (FP32 sums of at most 128 terms near 1 are good to 1e-4; so may ties be)
    assert (logits.gather(1, ids) - logits.topk(2, 1).values).abs().max() < 1e-4
    names = ("pre", "post", "next", "w_gate", "w_up", "w_down")
    p = {name: getattr(block, name).double().cpu().requires_grad_() for name in names}
    x64 = x.double().cpu().requires_grad_()
    want_h, want_n = plain(block, x64, ids, weights, p)
    (want_h * dh.double().cpu()).sum().add((want_n * dn.double().cpu()).sum()).backward()

    base = x64.detach()
    assert relative(h - x, want_h.detach() - base) < 2.0 ** -6
    assert relative(n, want_n.detach()) < 2.0 ** -6
    assert relative(served - x, want_h.detach() - base) < 2.0 ** -3
    assert relative(grads["x"], x64.grad) < 2.0 ** -5
    for name in names:
        assert relative(grads[name], p[name].grad) < 2.0 ** -5, name
