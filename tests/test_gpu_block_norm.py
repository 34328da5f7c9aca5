"""block_norm and block_norm_backward against 64-bit results, value by value.

Bounds (u: half a unit in the last place of the type, v = 2^-23): a sum of D squares is
off by at most D v / 2 of itself whatever its order, so 1 / rms by (D / 4 + 4) v; a value of
h by the FP32 steps before its rounding, eight half units of the magnitudes that are
added; the gradients likewise by their formulas' terms, and column sums of T tokens by T v of
the sum of magnitudes.
"""
from __future__ import annotations

import pytest
import torch

import raggedroute_amd as rr
from block_helpers import CODES, LEAST, ROUNDING, TYPES, Buf, assert_within, context

pytestmark = pytest.mark.gpu
V = 2.0 ** -23
SCALE, EPS = 0.7, 1e-5


def make(t, d, dtype, block_dtype, gate_tokens, post=True, block=True, seed=0):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dt=dtype):
        return torch.randn(*shape, device="cuda:0", generator=gen).mul_(std).add_(mean).to(TYPES[dt])

    v = {"x": normal(t, d, std=2.0), "pre_weight": normal(d, std=0.2, mean=1.0), "dh": normal(t, d), "dn": normal(t, d)}
    if block:
        v["block"] = normal(t, d, dt=block_dtype)
        if post:
            v["post_weight"] = normal(d, std=0.2, mean=1.0)
        if gate_tokens:
            v["gate"] = normal((t + gate_tokens - 1) // gate_tokens, d, std=0.5, mean=0.5)
    return v


def call(v, names, out, t, d, dtype, block_dtype, gate_tokens, cls, entry, size, offset=0):
    bufs = {name: Buf(v[name], offset=offset) for name in names if name in v}
    args = cls(**{name: b.ptr for name, b in {**bufs, **out}.items()}, residual_scale=SCALE, eps=EPS,
               gate_tokens=gate_tokens, tokens=t, hidden=d, dtype=CODES[dtype], block_dtype=CODES[block_dtype])
    ctx, ws = context(size(args))
    status = entry(args, ctx)
    assert status.ok(), status.message
    for name, b in {**bufs, **out, "workspace": ws}.items():
        assert b.intact(), f"{name}: written outside"
    return {name: b.t for name, b in out.items()}


def forward(v, t, d, dtype, block_dtype, gate_tokens, offset=0, outputs=("h", "n")):
    out = {name: Buf(shape=(t, d), dtype=TYPES[dtype], offset=offset) for name in outputs}
    return call(v, ("x", "block", "post_weight", "gate", "pre_weight"), out, t, d, dtype, block_dtype, gate_tokens,
                rr.BlockNormArgs, rr.block_norm, rr.get_block_norm_workspace_size, offset)


def terms(v, gate_tokens):
    """gate rows a token, N(block) or block, 1 / rms(block) in 64 bits."""
    block = v["block"].double()
    gate = v["gate"].double().repeat_interleave(gate_tokens, 0)[:block.shape[0]] if "gate" in v else torch.ones_like(block)
    if "post_weight" not in v:
        return gate, block, torch.ones(block.shape[0], 1, device="cuda:0", dtype=torch.float64)
    r = (block.square().mean(1, keepdim=True) + EPS).rsqrt()
    return gate, block * r * v["post_weight"].double(), r


def check_forward(v, got, dtype, gate_tokens):
    d = v["x"].shape[1]
    u, least, er = ROUNDING[dtype], LEAST[dtype], (d / 4 + 4) * V
    x = v["x"].double()
    h, eh = x, torch.zeros_like(x)
    if "block" in v:
        gate, b, _ = terms(v, gate_tokens)
        b = SCALE * gate * b
        h = x + b
        eh = (er + 8 * V) * b.abs() + 2 * V * h.abs()
    if "h" in got:
        assert_within(got["h"], h, eh * (1 + u) + u * h.abs() + least, "h")
    if "n" in got:
        r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
        w = v["pre_weight"].double()
        n = h * r * w
        # 1 / rms moves with the errors of h: by at most their 2-norm over h's
        moved = eh.square().sum(1, keepdim=True).sqrt() / h.square().sum(1, keepdim=True).sqrt().clamp_min(1e-300)
        en = (eh * r * w.abs()) + (er + 4 * V + moved) * n.abs()
        assert_within(got["n"], n, en * (1 + u) + u * n.abs() + least, "n")


TYPE_PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]


@pytest.mark.parametrize("dtype,block_dtype", TYPE_PAIRS)
@pytest.mark.parametrize("t,d,gate_tokens", [(1, 1, 1), (3, 7, 2), (5, 64, 0), (9, 513, 4), (2, 1024, 1), (4, 1030, 3),
                                             (3, 4096, 2), (2, 8191, 0), (3, 16384, 1), (2, 17001, 2), (700, 96, 50)])
def test_forward(device, t, d, gate_tokens, dtype, block_dtype):
    v = make(t, d, dtype, block_dtype, gate_tokens, seed=t * d)
    check_forward(v, forward(v, t, d, dtype, block_dtype, gate_tokens), dtype, gate_tokens)


@pytest.mark.parametrize("d", [264, 1001, 20000])
@pytest.mark.parametrize("post,block,outputs", [(False, True, ("h", "n")), (True, False, ("h", "n")), (True, False, ("n",)),
                                                (True, True, ("h",))])
def test_forward_without_parts(device, d, post, block, outputs):
    v = make(6, d, "bf16", "bf16", 2, post=post, block=block, seed=d)
    check_forward(v, forward(v, 6, d, "bf16", "bf16", 2, offset=1, outputs=outputs), "bf16", 2)


def backward(v, t, d, dtype, block_dtype, gate_tokens, offset=0, skip=()):
    out = {"dx": Buf(shape=(t, d), dtype=TYPES[dtype], offset=offset),
           "dpre_weight": Buf(shape=(d,), dtype=TYPES[dtype], offset=offset)}
    if "block" in v:
        out["dblock"] = Buf(shape=(t, d), dtype=TYPES[block_dtype], offset=offset)
        if "post_weight" in v:
            out["dpost_weight"] = Buf(shape=(d,), dtype=TYPES[dtype], offset=offset)
        if "gate" in v:
            out["dgate"] = Buf(shape=v["gate"].shape, dtype=TYPES[dtype], offset=offset)
    out = {name: b for name, b in out.items() if name not in skip}
    return call(v, ("h", "block", "post_weight", "gate", "pre_weight", "dh", "dn"), out, t, d, dtype, block_dtype,
                gate_tokens, rr.BlockNormBackwardArgs, rr.block_norm_backward, rr.get_block_norm_backward_workspace_size,
                offset)


def check_backward(v, got, dtype, block_dtype, gate_tokens):
    t, d = v["h"].shape
    u, least, er = ROUNDING[dtype], LEAST[dtype], (d / 4 + 4) * V
    h = v["h"].double()
    dx = v["dh"].double() if "dh" in v else torch.zeros_like(h)
    edx = torch.zeros_like(dx)
    rounded = lambda want, err, ut=u, lt=least: err * (1 + ut) + ut * want.abs() + lt  # noqa: E731
    pre, epre = torch.zeros_like(h), torch.zeros_like(h)
    if "dn" in v:
        r = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
        w, dn = v["pre_weight"].double(), v["dn"].double()
        back = (dn * w * h).mean(1, keepdim=True) * r * r
        eback = (d * V + 2 * er + 8 * V) * (dn * w * h).abs().mean(1, keepdim=True) * r * r
        dx = dx + r * (dn * w - h * back)
        edx = r * ((er + 8 * V) * ((dn * w).abs() + (h * back).abs()) + h.abs() * eback) + 4 * V * (dx.abs() + 1)
        pre, epre = dn * h * r, (er + 4 * V) * (dn * h * r).abs()
    assert_within(got["dx"], dx, rounded(dx, edx), "dx")

    def column(name, value, err, groups=None):
        if name not in got:
            return
        total, size = value, err + 2 * t * V * value.abs()
        if groups is None:
            total, size = total.sum(0), size.sum(0)
        else:
            rows = torch.arange(t, device="cuda:0") // groups
            zero = torch.zeros(v["gate"].shape, dtype=torch.float64, device="cuda:0")
            total, size = zero.index_add(0, rows, total), zero.index_add(0, rows, size)
        assert_within(got[name], total, rounded(total, size), name)

    column("dpre_weight", pre, epre)
    if "block" not in v:
        return
    gate, b, rb = terms(v, gate_tokens)
    unit = v["block"].double() * rb
    eb = (er + 4 * V) * b.abs() if "post_weight" in v else torch.zeros_like(b)
    column("dgate", SCALE * dx * b, SCALE * (edx * b.abs() + dx.abs() * eb) + 4 * V * (dx * b).abs(), gate_tokens)
    db = SCALE * gate * dx
    edb = SCALE * gate.abs() * edx + 4 * V * db.abs()
    column("dpost_weight", db * unit, edb * unit.abs() + (er + 4 * V) * (db * unit).abs())
    if "dblock" in got:
        ub, lb = ROUNDING[block_dtype], LEAST[block_dtype]
        if "post_weight" in v:
            w = v["post_weight"].double()
            back = (db * w * unit).mean(1, keepdim=True)
            eback = ((edb * (w * unit).abs()) + (d * V + er + 8 * V) * (db * w * unit).abs()).mean(1, keepdim=True)
            want = rb * (db * w - unit * back)
            err = rb * (edb * w.abs() + (2 * er + 8 * V) * ((db * w).abs() + (unit * back).abs()) + unit.abs() * eback)
        else:
            want, err = db, edb
        assert_within(got["dblock"], want, rounded(want, err + 4 * V * want.abs(), ub, lb), "dblock")


# gate rows of one token, of a few, of more than a workgroup takes, none; ragged last ones
BACKWARD = [(1, 1, 1), (3, 7, 2), (5, 64, 0), (9, 513, 4), (4, 1030, 3), (3, 4096, 2), (2, 8191, 0), (3, 16384, 1),
            (5, 17001, 2), (1500, 96, 700), (2500, 520, 1), (5000, 264, 7), (3000, 1024, 3000), (700, 4000, 64)]


@pytest.mark.parametrize("dtype,block_dtype", TYPE_PAIRS)
@pytest.mark.parametrize("t,d,gate_tokens", BACKWARD)
def test_backward(device, t, d, gate_tokens, dtype, block_dtype):
    v = make(t, d, dtype, block_dtype, gate_tokens, seed=t + d)
    v["h"] = v.pop("x")
    check_backward(v, backward(v, t, d, dtype, block_dtype, gate_tokens), dtype, block_dtype, gate_tokens)


@pytest.mark.parametrize("d", [264, 1001, 20000])
@pytest.mark.parametrize("post,block,drop", [(False, True, ()), (True, False, ()), (True, True, ("dh",)), (True, True, ("dn",))])
def test_backward_without_parts(device, d, post, block, drop):
    v = make(40, d, "bf16", "bf16", 3, post=post, block=block, seed=d)
    v["h"] = v.pop("x")
    for name in drop:
        v.pop(name)
    check_backward(v, backward(v, 40, d, "bf16", "bf16", 3, offset=1), "bf16", "bf16", 3)


@pytest.mark.parametrize("skip", [("dblock",), ("dgate",), ("dpre_weight",), ("dpost_weight",),
                                  ("dblock", "dgate", "dpre_weight", "dpost_weight")])
@pytest.mark.parametrize("gate_tokens", [1, 30])
def test_backward_unwanted(device, skip, gate_tokens):
    v = make(60, 520, "f16", "f16", gate_tokens, seed=1)
    v["h"] = v.pop("x")
    check_backward(v, backward(v, 60, 520, "f16", "f16", gate_tokens, skip=skip), "f16", "f16", gate_tokens)


def test_in_place(device):
    """h may be x, dx may be dh, dblock may be block."""
    t, d = 33, 1030
    for width in (d, 20002):
        v = make(t, width, "bf16", "bf16", 4, seed=2)
        want = forward(v, t, width, "bf16", "bf16", 4)
        x, n = Buf(v["x"]), Buf(shape=(t, width), dtype=torch.bfloat16)
        b = {name: Buf(v[name]) for name in ("block", "post_weight", "gate", "pre_weight")}
        common = dict(residual_scale=SCALE, eps=EPS, gate_tokens=4, tokens=t, hidden=width)
        ctx, _ = context()
        assert rr.block_norm(rr.BlockNormArgs(x=x.ptr, h=x.ptr, n=n.ptr, **{k: q.ptr for k, q in b.items()}, **common), ctx).ok()
        assert torch.equal(x.t, want["h"]) and torch.equal(n.t, want["n"])
        v["h"] = v.pop("x")
        want = backward(v, t, width, "bf16", "bf16", 4)
        h, dh, dn = Buf(v["h"]), Buf(v["dh"]), Buf(v["dn"])
        args = rr.BlockNormBackwardArgs(h=h.ptr, dh=dh.ptr, dn=dn.ptr, dx=dh.ptr, dblock=b["block"].ptr,
                                        **{k: q.ptr for k, q in b.items()}, **common)
        ctx, _ = context(rr.get_block_norm_backward_workspace_size(args))
        assert rr.block_norm_backward(args, ctx).ok()
        assert torch.equal(dh.t, want["dx"]) and torch.equal(b["block"].t, want["dblock"])


def test_gradients_against_differences(device):
    """FP32 gradients along random directions against central differences of the 64-bit
    formula: step 1e-5, good to about 1e-7 of the sum of magnitudes."""
    t, d, every = 13, 72, 5
    v = make(t, d, "f32", "f32", every, seed=3)
    got = forward(v, t, d, "f32", "f32", every)
    w = {**v, "h": got["h"]}
    w.pop("x")
    grad = backward(w, t, d, "f32", "f32", every)
    base = {name: v[name].double() for name in ("x", "block", "post_weight", "gate", "pre_weight")}

    def loss(p):
        b = p["block"] * (p["block"].square().mean(1, keepdim=True) + EPS).rsqrt() * p["post_weight"]
        h = p["x"] + SCALE * p["gate"].repeat_interleave(every, 0)[:t] * b
        n = h * (h.square().mean(1, keepdim=True) + EPS).rsqrt() * p["pre_weight"]
        return (h * v["dh"].double()).sum() + (n * v["dn"].double()).sum()

    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(0)
    for name in base:
        step = torch.randn(base[name].shape, device="cuda:0", generator=gen, dtype=torch.float64)
        eps = 1e-5
        diff = (loss({**base, name: base[name] + eps * step}) - loss({**base, name: base[name] - eps * step})) / (2 * eps)
        g = grad["d" + name].double()
        assert abs((g * step).sum() - diff) <= 2e-6 * (g * step).abs().sum() + 1e-7, name


def test_special_rows(device):
    """A zero row stays zero, a row with a NaN or infinity spoils only itself."""
    t, d = 6, 200
    v = make(t, d, "bf16", "bf16", 0, seed=4)
    v["x"][0], v["block"][0] = 0.0, 0.0
    v["block"][2, 7], v["x"][4, 0] = float("nan"), float("inf")
    got = forward(v, t, d, "bf16", "bf16", 0)
    assert (got["h"][0] == 0).all() and (got["n"][0] == 0).all()
    assert torch.isnan(got["n"][2]).all() and not torch.isfinite(got["n"][4]).all()
    assert torch.isfinite(got["n"][[0, 1, 3, 5]]).all()


def test_equal_calls_give_equal_bits_and_no_tokens(device):
    v = make(900, 1000, "bf16", "bf16", 300, seed=5)
    v["h"] = v.pop("x")
    first, again = (backward(v, 900, 1000, "bf16", "bf16", 300) for _ in range(2))
    assert all(torch.equal(first[name], again[name]) for name in first)
    none = make(0, 64, "bf16", "bf16", 0)
    none["h"] = none.pop("x")
    got = backward(none, 0, 64, "bf16", "bf16", 0)
    assert (got["dpre_weight"] == 0).all() and (got["dpost_weight"] == 0).all()
