"""gated_ffn and gated_ffn_backward against 64-bit results, value by value.

Bounds (u: half a unit in the last place of the type; FP32 sums of n products are off by
at most n 2^-23 of the sum of their magnitudes, in any order): e(g) = K 2^-23 |x||Wg|,
likewise u; a = act(g) u is off by |act'| <= 1.2 times e(g)|u| + |act(g)| e(u), 2^-20 of itself
for the exponential, and u for its rounding; y by its own rounding, the sums and e(a)|Wd|.
The backward pass starts from rounded gate, up and act (inputs here), its bounds follow its
formulas in the same way.
"""
from __future__ import annotations

import pytest
import torch

import raggedroute_amd as rr
from block_helpers import (ACTIVATIONS, CODES, LEAST, ROUNDING, TYPES, Buf, assert_within, context, offsets_of,
                           segments)

pytestmark = pytest.mark.gpu

FAMILIES = {"auto": rr.kernel(), "naive": rr.kernel(rr.KernelFamily.kNaive)}
SUM = 2.0 ** -23
EXP = 2.0 ** -20


def make(counts, k, f, n, dtype, seed=0, offset=0):
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda:0", generator=gen).mul_(std).to(TYPES[dtype])

    offs, rows = offsets_of(counts)
    e = len(counts)
    v = {"x": normal(rows, k), "w_gate": normal(e, k, f, std=k ** -0.5), "w_up": normal(e, k, f, std=k ** -0.5),
         "w_down": normal(e, f, n, std=f ** -0.5), "dy": normal(rows, n), "gate": normal(rows, f),
         "up": normal(rows, f), "act": normal(rows, f)}
    b = {name: Buf(t, offset=offset) for name, t in v.items()}
    b["offsets"] = Buf(offs)
    return v, b, rows


def forward(b, counts, rows, k, f, n, dtype, act="silu", keep=True, y_dtype=None, family="auto", offset=0):
    y_dtype = y_dtype or dtype
    out = {name: Buf(shape=(rows, f), dtype=TYPES[dtype], offset=offset) for name in ("gate", "up", "act")}
    out["y"] = Buf(shape=(rows, n), dtype=TYPES[y_dtype], offset=offset)
    args = rr.GatedFfnArgs(x=b["x"].ptr, w_gate=b["w_gate"].ptr, w_up=b["w_up"].ptr, w_down=b["w_down"].ptr,
                           offsets=b["offsets"].ptr, gate=out["gate"].ptr if keep else None,
                           up=out["up"].ptr if keep else None, act=out["act"].ptr, y=out["y"].ptr, rows=rows,
                           experts=len(counts), hidden=k, inner=f, output=n,
                           activation=int(ACTIVATIONS[act][0]), dtype=CODES[dtype], y_dtype=CODES[y_dtype],
                           kernel=FAMILIES[family])
    ctx, ws = context(rr.get_gated_ffn_workspace_size(args))
    status = rr.gated_ffn(args, ctx)
    assert status.ok(), status.message
    for name, buf in {**b, **out, "workspace": ws}.items():
        assert buf.intact(), f"{name}: written outside"
    return out


def check_forward(v, out, counts, dtype, act, keep=True, y_dtype=None):
    u, least = ROUNDING[dtype], LEAST[dtype]
    uy, ly = ROUNDING[y_dtype or dtype], LEAST[y_dtype or dtype]
    fn = ACTIVATIONS[act][1]
    k, f = v["w_gate"].shape[1:]
    got = {name: out[name].t for name in out}
    for e, rows in segments(counts):
        x, wg, wu, wd = (t.double() for t in (v["x"][rows], v["w_gate"][e], v["w_up"][e], v["w_down"][e]))
        g, up = x @ wg, x @ wu
        eg, eu = k * SUM * (x.abs() @ wg.abs()), k * SUM * (x.abs() @ wu.abs())
        if keep:
            assert_within(got["gate"][rows], g, eg + u * g.abs() + least, "gate")
            assert_within(got["up"][rows], up, eu + u * up.abs() + least, "up")
        a = fn(g) * up
        ea = 1.2 * eg * (up.abs() + eu) + fn(g).abs() * eu + (EXP + u) * 1.01 * a.abs() + least
        assert_within(got["act"][rows], a, ea, "act")
        y = a @ wd
        sums = f * SUM * ((a.abs() + ea) @ wd.abs())
        assert_within(got["y"][rows], y, uy * y.abs() + (ea @ wd.abs() + sums) * (1 + uy) + ly, "y")


# experts with no rows at both ends and between, one row, tiles that end inside and on their edge
SHAPES = [
    ([1], 1, 1, 1),
    ([3, 0, 1], 2, 3, 5),
    ([0, 5, 0, 0, 17, 1, 0], 33, 65, 47),
    ([16, 16, 15], 64, 32, 64),
    ([0, 0, 2], 128, 256, 128),
    ([1, 1, 0, 1, 4], 256, 96, 264),
    ([70, 0, 31], 72, 136, 200),
    ([129, 64, 1, 127], 136, 129, 130),
    ([256, 300, 0, 12], 96, 264, 72),
    ([513], 200, 131, 257),
    ([40] * 9, 320, 192, 320),
]


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("dtype,act", [("bf16", "silu"), ("f16", "gelu")])
@pytest.mark.parametrize("counts,k,f,n", SHAPES)
def test_forward(device, counts, k, f, n, dtype, act, family):
    v, b, rows = make(counts, k, f, n, dtype)
    check_forward(v, forward(b, counts, rows, k, f, n, dtype, act, family=family), counts, dtype, act)


@pytest.mark.parametrize("counts,k,f,n", [([9, 0, 200], 96, 136, 72), ([2, 1], 33, 17, 31), ([1, 0, 3], 512, 256, 512)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_forward_serving_types_and_alignment(device, counts, k, f, n, offset):
    """Without gate and up, FP32 results, and buffers off every vector boundary."""
    v, b, rows = make(counts, k, f, n, "bf16", offset=offset)
    out = forward(b, counts, rows, k, f, n, "bf16", keep=False, y_dtype="f32", offset=offset)
    check_forward(v, out, counts, "bf16", "silu", keep=False, y_dtype="f32")
    assert out["gate"].untouched(slice(None)) and out["up"].untouched(slice(None))


@pytest.mark.parametrize("rows_each,k,f,n", [(1, 1024, 512, 1024), (5, 1000, 344, 500), (33, 512, 1024, 512),
                                             (150, 264, 520, 1032), (700, 1024, 512, 512)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_forward_longer_sums(device, rows_each, k, f, n, dtype):
    counts = [rows_each, 0, rows_each + 3, 2 * rows_each]
    v, b, rows = make(counts, k, f, n, dtype, seed=3)
    check_forward(v, forward(b, counts, rows, k, f, n, dtype), counts, dtype, "silu")


def backward(b, counts, rows, k, f, n, dtype, act="silu", family="auto", offset=0, skip=()):
    shapes = {"dx": (rows, k), "dw_gate": (len(counts), k, f), "dw_up": (len(counts), k, f),
              "dw_down": (len(counts), f, n)}
    out = {name: Buf(shape=s, dtype=TYPES[dtype], offset=offset) for name, s in shapes.items() if name not in skip}
    args = rr.GatedFfnBackwardArgs(
        **{name: b[name].ptr for name in ("x", "w_gate", "w_up", "w_down", "offsets", "gate", "up", "act", "dy")},
        **{name: buf.ptr for name, buf in out.items()}, rows=rows, experts=len(counts), hidden=k, inner=f, output=n,
        activation=int(ACTIVATIONS[act][0]), dtype=CODES[dtype], kernel=FAMILIES[family])
    ctx, ws = context(rr.get_gated_ffn_backward_workspace_size(args))
    status = rr.gated_ffn_backward(args, ctx)
    assert status.ok(), status.message
    for name, buf in {**b, **out, "workspace": ws}.items():
        assert buf.intact(), f"{name}: written outside"
    return out


def grads(v, counts, e, rows, dtype, act):
    """64-bit gradients of one expert and their bounds."""
    u, least = ROUNDING[dtype], LEAST[dtype]
    f, n = v["w_down"].shape[1:]
    x, wg, wu, wd, dy, gate, up, a = (t.double() for t in (
        v["x"][rows], v["w_gate"][e], v["w_up"][e], v["w_down"][e], v["dy"][rows], v["gate"][rows], v["up"][rows],
        v["act"][rows]))
    g = gate.clone().requires_grad_()
    s = ACTIVATIONS[act][1](g)
    slope = torch.autograd.grad(s.sum(), g)[0] if g.numel() else torch.zeros_like(g)
    s = s.detach()
    da = dy @ wd.t()
    eda = n * SUM * (dy.abs() @ wd.abs().t())
    dg, du = da * up * slope, da * s
    eslope = EXP * (1.0 + gate.abs())
    edg = (da.abs() + eda) * up.abs() * eslope + eda * (up * slope).abs() + u * 1.01 * dg.abs() + least
    edu = (da.abs() + eda) * s.abs() * EXP + eda * s.abs() + u * 1.01 * du.abs() + least
    ag, au = dg.abs() + edg, du.abs() + edu
    r = x.shape[0]
    want = {"dx": dg @ wg.t() + du @ wu.t(), "dw_gate": x.t() @ dg, "dw_up": x.t() @ du, "dw_down": a.t() @ dy}
    bound = {"dx": edg @ wg.abs().t() + edu @ wu.abs().t() + 2 * f * SUM * (ag @ wg.abs().t() + au @ wu.abs().t()),
             "dw_gate": x.abs().t() @ edg + r * SUM * (x.abs().t() @ ag),
             "dw_up": x.abs().t() @ edu + r * SUM * (x.abs().t() @ au),
             "dw_down": r * SUM * (a.abs().t() @ dy.abs())}
    return want, {name: (1 + u) * t + u * want[name].abs() + least for name, t in bound.items()}


def check_backward(v, out, counts, dtype, act):
    got = {name: buf.t for name, buf in out.items()}
    for e, rows in segments(counts):
        want, bound = grads(v, counts, e, rows, dtype, act)
        for name in got:
            assert_within(got[name][rows if name == "dx" else e], want[name], bound[name], f"{name} of expert {e}")


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("dtype,act", [("bf16", "gelu"), ("f16", "silu")])
@pytest.mark.parametrize("counts,k,f,n", SHAPES)
def test_backward(device, counts, k, f, n, dtype, act, family):
    v, b, rows = make(counts, k, f, n, dtype, seed=1)
    check_backward(v, backward(b, counts, rows, k, f, n, dtype, act, family), counts, dtype, act)


@pytest.mark.parametrize("counts,k,f,n", [([9, 0, 200], 96, 136, 72), ([2, 1], 33, 17, 31)])
@pytest.mark.parametrize("offset", [1, 4])
def test_backward_alignment(device, counts, k, f, n, offset):
    v, b, rows = make(counts, k, f, n, "f16", seed=2, offset=offset)
    check_backward(v, backward(b, counts, rows, k, f, n, "f16", "silu", offset=offset), counts, "f16", "silu")


@pytest.mark.parametrize("counts,k,f,n", [([700, 0, 300], 1024, 512, 512), ([1, 40, 2], 520, 264, 1000)])
def test_backward_longer_sums(device, counts, k, f, n):
    v, b, rows = make(counts, k, f, n, "bf16", seed=4)
    check_backward(v, backward(b, counts, rows, k, f, n, "bf16", "silu"), counts, "bf16", "silu")


@pytest.mark.parametrize("k,f,n", [(2048, 40, 72), (40, 264, 17), (256, 128, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_few_rows_and_a_long_expert(device, k, f, n, dtype):
    """Few rows an expert on average, but one expert with more than a block of them."""
    counts = [0, 37, 0, 1, 2] + [0] * 7
    v, b, rows = make(counts, k, f, n, dtype, seed=12)
    check_forward(v, forward(b, counts, rows, k, f, n, dtype), counts, dtype, "silu")


@pytest.mark.parametrize("counts,k,f,n", [([256, 0, 600], 264, 136, 392), ([257, 511, 300], 64, 520, 72),
                                          ([1000], 200, 264, 128)])
@pytest.mark.parametrize("dtype,act", [("bf16", "silu"), ("f16", "gelu")])
def test_many_rows_an_expert(device, counts, k, f, n, dtype, act):
    """Segments on both sides of 256 rows and of its cuts, slices and columns that end inside."""
    v, b, rows = make(counts, k, f, n, dtype, seed=11)
    check_forward(v, forward(b, counts, rows, k, f, n, dtype, act), counts, dtype, act)
    check_backward(v, backward(b, counts, rows, k, f, n, dtype, act), counts, dtype, act)


@pytest.mark.parametrize("skip", [("dx",), ("dw_gate", "dw_up"), ("dw_down",), ("dx", "dw_down")])
def test_backward_unwanted_gradients(device, skip):
    counts, k, f, n = [20, 0, 9], 72, 40, 64
    v, b, rows = make(counts, k, f, n, "bf16", seed=5)
    check_backward(v, backward(b, counts, rows, k, f, n, "bf16", skip=skip), counts, "bf16", "silu")


@pytest.mark.parametrize("family", ["auto", "naive"])
def test_no_rows(device, family):
    """Forward writes nothing; the weight gradients are zero."""
    counts, k, f, n = [0, 0, 0], 40, 24, 16
    v, b, rows = make(counts, k, f, n, "bf16")
    forward(b, counts, rows, k, f, n, "bf16", family=family)
    out = backward(b, counts, rows, k, f, n, "bf16", family=family)
    for name in ("dw_gate", "dw_up", "dw_down"):
        assert (out[name].t == 0).all()


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("counts,k,f,n", [([3, 0, 5], 72, 40, 64), ([140, 0, 5], 33, 65, 47)])
def test_neighbours_do_not_leak(device, counts, k, f, n, family):
    """Infinities and NaN in another expert's weights and rows, and rows past the last
    segment, reach no result of the others; those rows are left alone."""
    v, b, rows = make(counts + [4], k, f, n, "bf16", seed=6)
    clean = sum(counts)
    for name in ("x", "dy", "gate", "up", "act"):
        v[name][clean:] = float("nan")
    for name in ("w_gate", "w_up", "w_down"):
        v[name][1] = float("inf")
        v[name][-1] = float("nan")
    b = {name: Buf(t) for name, t in v.items()}
    b["offsets"] = Buf(offsets_of(counts + [0])[0])
    every = counts + [0]
    out = forward(b, every, rows, k, f, n, "bf16", family=family)
    check_forward(v, out, counts, "bf16", "silu")
    for name in out:
        assert out[name].untouched(slice(clean, None)), name
    grad = backward(b, every, rows, k, f, n, "bf16", family=family)
    assert grad["dx"].untouched(slice(clean, None))
    assert (grad["dw_gate"].t[1] == 0).all() and (grad["dw_down"].t[-1] == 0).all()
    for e, seg in segments(counts):
        want, bound = grads(v, counts, e, seg, "bf16", "silu")
        if seg.stop > seg.start:
            assert_within(grad["dx"].t[seg], want["dx"], bound["dx"], "dx")
            for name in ("dw_gate", "dw_up", "dw_down"):
                assert_within(grad[name].t[e], want[name], bound[name], name)


def test_nan_and_infinity_stay_in_their_row(device):
    counts, k, f, n = [6, 150], 64, 128, 64
    v, b, rows = make(counts, k, f, n, "bf16", seed=7)
    v["x"][2, 5] = float("nan")
    v["x"][40, 0] = float("inf")
    b["x"] = Buf(v["x"])
    y = forward(b, counts, rows, k, f, n, "bf16")["y"].t
    bad = ~torch.isfinite(y)
    assert bad[2].all() and bad[40].any()
    bad[2] = bad[40] = False
    assert not bad.any()


def test_large_preactivations(device):
    """act at preactivations past every exponent: 0 or the value itself, slopes 0 or 1."""
    counts, k, f, n = [7], 1, 8, 8
    v, b, rows = make(counts, k, f, n, "bf16", seed=8)
    values = torch.tensor([-3e38, -1e20, -100.0, 0.0, 100.0, 1e20, 3e38], device="cuda:0")
    gate = values[:, None].expand(7, f)
    v["gate"], v["up"] = gate.to(torch.bfloat16).contiguous(), torch.ones(7, f, device="cuda:0", dtype=torch.bfloat16)
    v["dy"] = torch.zeros_like(v["dy"])
    v["dy"][:, 0] = 1.0
    v["w_down"] = torch.zeros_like(v["w_down"])
    v["w_down"][0, :, 0] = 1.0
    v["w_gate"], v["w_up"] = torch.ones_like(v["w_gate"]), torch.zeros_like(v["w_up"])
    b = {**b, **{name: Buf(v[name]) for name in ("gate", "up", "dy", "w_down", "w_gate", "w_up")}}
    for act in ACTIVATIONS:
        dx = backward(b, counts, rows, k, f, n, "bf16", act)["dx"].t.double().flatten()
        want = torch.tensor([0, 0, 0, 0.5, 1, 1, 1], dtype=torch.float64, device="cuda:0") * f
        assert torch.equal(dx, want), (act, dx)


@pytest.mark.parametrize("counts,k,f,n", [([5, 0, 9], 24, 40, 16), ([130, 64], 64, 72, 96)])
def test_equal_calls_give_equal_bits(device, counts, k, f, n):
    v, b, rows = make(counts, k, f, n, "bf16", seed=9)
    first = {**forward(b, counts, rows, k, f, n, "bf16"), **backward(b, counts, rows, k, f, n, "bf16")}
    again = {**forward(b, counts, rows, k, f, n, "bf16"), **backward(b, counts, rows, k, f, n, "bf16")}
    for name in first:
        assert torch.equal(first[name].t.view(torch.uint8), again[name].t.view(torch.uint8)), name


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_against_differences(device, act):
    """The gradients along random directions against central differences of the 64-bit
    block, from a forward pass of the kernels. The differences (step 1e-4) are good to
    1e-6; the gradients' own error is that of rounding g, u and a (u each, entering every
    gradient once) and of the results, four roundings in all."""
    counts, k, f, n = [5, 0, 40], 24, 40, 32
    v, b, rows = make(counts, k, f, n, "f16", seed=10)
    out = forward(b, counts, rows, k, f, n, "f16", act)
    grad = backward({**b, "gate": out["gate"], "up": out["up"], "act": out["act"]}, counts, rows, k, f, n, "f16", act)
    base = {name: v[name].double() for name in ("x", "w_gate", "w_up", "w_down")}
    dy, fn = v["dy"].double(), ACTIVATIONS[act][1]

    def loss(t):
        total = 0.0
        for e, seg in segments(counts):
            y = (fn(t["x"][seg] @ t["w_gate"][e]) * (t["x"][seg] @ t["w_up"][e])) @ t["w_down"][e]
            total = total + (y * dy[seg]).sum()
        return total

    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(0)
    for name in base:
        got = grad["d" + name].t.double()
        step = torch.randn(base[name].shape, device="cuda:0", generator=gen, dtype=torch.float64)
        h = 1e-4
        diff = (loss({**base, name: base[name] + h * step}) - loss({**base, name: base[name] - h * step})) / (2 * h)
        size = (got.square() * step.square()).sum().sqrt()  # spread of the sum's independent errors, per unit
        assert abs((got * step).sum() - diff) <= (4 * ROUNDING["f16"] * 6) * size + 1e-6 * abs(diff), name


def test_other_stream_and_graph(device):
    """On a stream of its own, and replayed from a graph with new inputs between replays."""
    counts, k, f, n = [12, 0, 140, 3], 64, 72, 80
    stream = torch.cuda.Stream()
    v, b, rows = make(counts, k, f, n, "bf16", seed=11)
    offs, _ = offsets_of(counts)
    x, wg, wu, wd = v["x"].clone(), v["w_gate"], v["w_up"], v["w_down"]
    act = torch.zeros(rows, f, dtype=torch.bfloat16, device="cuda:0")
    y = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda:0")
    args = rr.GatedFfnArgs(x=x.data_ptr(), w_gate=wg.data_ptr(), w_up=wu.data_ptr(), w_down=wd.data_ptr(),
                           offsets=offs.data_ptr(), act=act.data_ptr(), y=y.data_ptr(), rows=rows,
                           experts=len(counts), hidden=k, inner=f, output=n)
    torch.cuda.synchronize()
    ctx, _ = context(stream=stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        assert rr.gated_ffn(args, ctx).ok()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert rr.gated_ffn(args, rr.RuntimeContext(stream=torch.cuda.current_stream().cuda_stream,
                                                        architecture=ctx.architecture)).ok()
    for seed in range(3):
        fresh = make(counts, k, f, n, "bf16", seed=20 + seed)[0]["x"]
        x.copy_(fresh)
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = y.clone()
        with torch.cuda.stream(stream):
            assert rr.gated_ffn(args, ctx).ok()
        torch.cuda.synchronize()
        assert torch.equal(replayed, y) and (y != 0).any()


@pytest.mark.parametrize("counts,k,f,n", [([1], 2048, 40, 24), ([2, 0, 1], 3000, 2100, 130), ([0, 3], 260, 4100, 17),
                                          ([17], 2304, 8, 8), ([20, 0, 30], 2048, 2048, 48)])
@pytest.mark.parametrize("dtype,y_dtype", [("bf16", "bf16"), ("f16", "f32")])
def test_forward_split_sums(device, counts, k, f, n, dtype, y_dtype):
    """Few rows of few wide experts: sums split over workgroups, parts in the workspace."""
    v, b, rows = make(counts, k, f, n, dtype, seed=12)
    check_forward(v, forward(b, counts, rows, k, f, n, dtype, y_dtype=y_dtype), counts, dtype, "silu", y_dtype=y_dtype)
