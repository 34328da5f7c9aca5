"""Gate, sort, experts, combine and their gradients as a training step runs them, the 4-bit operators
as a decode step runs them, captured graphs, other streams, and sizes past 32-bit offsets."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import raggedroute_amd as rr
from block_helpers import CODES, Buf, assert_within
from test_gpu_block_offsets import OFFSETS, bounds
from test_gpu_mxfp4 import encode, layout, pack, product, values, weights
from test_gpu_tokens import maps

pytestmark = pytest.mark.gpu
GFX950 = int(rr.DeviceArchitecture.kGfx950)


class Calls:
    """Calls with the workspace each asks for, run in order on a stream."""

    def __init__(self):
        self.calls, self.keep = [], []

    def add(self, name, args):
        size = getattr(rr, f"get_{name}_workspace_size")(args)
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda:0")
        self.keep.append(ws)
        self.calls.append((getattr(rr, name), args, ws.data_ptr(), size))

    def run(self, stream=None):
        stream = stream if stream is not None else torch.cuda.current_stream()
        for entry, args, ws, size in self.calls:
            status = entry(args, rr.RuntimeContext(stream=stream.cuda_stream, workspace=ws, workspace_bytes=size,
                                                   architecture=GFX950))
            assert status.ok(), status.message


def zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda:0")


def training_step(tokens, experts, hidden, inner, seed):
    """Inputs, outputs and calls of a step from logits and rows to every gradient."""
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (std * torch.randn(*shape, device="cuda:0", generator=gen)).to(dtype)

    rows = 2 * tokens
    t = dict(logits=normal(tokens, experts, dtype=torch.float32), x=normal(tokens, hidden, dtype=torch.float32),
             dy=normal(tokens, hidden, dtype=torch.float32), w_gate=normal(experts, hidden, inner, std=hidden ** -0.5),
             w_up=normal(experts, hidden, inner, std=hidden ** -0.5), w_down=normal(experts, inner, hidden, std=inner ** -0.5))
    f32, i32 = dict(dtype=torch.float32), dict(dtype=torch.int32)
    t |= dict(ids=zeros(tokens, 2, **i32), weights=zeros(tokens, 2, **f32), offsets=zeros(experts + 1, **i32),
              pos=zeros(rows, **i32), rows=zeros(rows, hidden), gate=zeros(rows, inner), up=zeros(rows, inner),
              act=zeros(rows, inner), r=zeros(rows, hidden), y=zeros(tokens, hidden, **f32), dr=zeros(rows, hidden),
              dweights=zeros(tokens, 2, **f32), dlogits=zeros(tokens, experts, **f32), drows=zeros(rows, hidden),
              dx=zeros(tokens, hidden, **f32), dw_gate=zeros(experts, hidden, inner), dw_up=zeros(experts, hidden, inner),
              dw_down=zeros(experts, inner, hidden))
    p = {name: v.data_ptr() for name, v in t.items()}
    bf16, fp32 = CODES["bf16"], CODES["f32"]
    calls = Calls()
    calls.keep.append(t)
    calls.add("topk_gate", rr.TopKGateArgs(logits=rr.cview(p["logits"]), expert_ids=p["ids"], weights=rr.mview(p["weights"]),
                                           tokens=tokens, experts=experts))
    calls.add("sort_tokens", rr.SortTokensArgs(x=p["x"], expert_ids=p["ids"], offsets=p["offsets"], route_pos=p["pos"],
                                               x_sorted=p["rows"], tokens=tokens, experts=experts, hidden=hidden,
                                               dtype=bf16, x_dtype=fp32))
    ffn = dict(x=p["rows"], w_gate=p["w_gate"], w_up=p["w_up"], w_down=p["w_down"], offsets=p["offsets"], gate=p["gate"],
               up=p["up"], act=p["act"], rows=rows, experts=experts, hidden=hidden, inner=inner, output=hidden, dtype=bf16)
    calls.add("gated_ffn", rr.GatedFfnArgs(y=p["r"], **ffn))
    both = dict(y_sorted=p["r"], route_pos=p["pos"], route_weights=p["weights"], tokens=tokens, hidden=hidden, dtype=bf16,
                y_dtype=fp32)
    calls.add("combine_tokens", rr.CombineTokensArgs(y=p["y"], **both))
    calls.add("combine_tokens_backward", rr.CombineTokensBackwardArgs(dy=p["dy"], dy_sorted=p["dr"],
                                                                      droute_weights=p["dweights"], **both))
    calls.add("topk_gate_backward", rr.TopKGateBackwardArgs(expert_ids=p["ids"], weights=p["weights"],
                                                            dweights=p["dweights"], dlogits=p["dlogits"], tokens=tokens,
                                                            experts=experts))
    calls.add("gated_ffn_backward", rr.GatedFfnBackwardArgs(dy=p["dr"], dx=p["drows"], dw_gate=p["dw_gate"],
                                                            dw_up=p["dw_up"], dw_down=p["dw_down"], **ffn))
    calls.add("sort_tokens_backward", rr.SortTokensBackwardArgs(dx_sorted=p["drows"], route_pos=p["pos"], dx=p["dx"],
                                                                tokens=tokens, hidden=hidden, dtype=bf16, x_dtype=fp32))
    return t, calls


def check_step(t):
    """Against 64 bits in norm: x's rounding to BF16 enters g, u and a (2^-9 of a value each, up to 1.5
    times as much through the activation), a's and r's own once more: under 5 * 2^-9 forward;
    backward the same for dr, dg, du, the kept g, u and a and the result: 2^-5. The logits' gradient
    is w1 w2 (<dy, r1> - <dy, r2>) and its negative: an error of r of 2^-6 of its norm moves a dot
    product by 2^-6 |dy| |r| at most (Cauchy and Schwarz), whatever the products cancel to, so that both
    entries are off by 2^-6 w1 w2 |dy| (|r1| + |r2|) at most."""
    v = {name: t[name].double().requires_grad_() for name in ("logits", "x", "w_gate", "w_up", "w_down")}
    ids = t["ids"].long()
    assert torch.equal(ids, t["logits"].topk(2, 1).indices)
    w = torch.softmax(v["logits"].gather(1, ids), 1)
    y = torch.zeros_like(v["x"])
    size = torch.zeros(ids.shape, dtype=torch.float64, device="cuda:0")  # |r|
    for e in range(t["logits"].shape[1]):
        token, rank = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            x = v["x"][token]
            r = (torch.nn.functional.silu(x @ v["w_gate"][e]) * (x @ v["w_up"][e])) @ v["w_down"][e]
            size[token, rank] = r.detach().norm(dim=1)
            y = y.index_add(0, token, w[token, rank][:, None] * r)
    grads = torch.autograd.grad(y, list(v.values()), t["dy"].double())

    def relative(got, want):
        return ((got.double() - want).norm() / want.norm()).item()

    assert relative(t["y"], y.detach()) < 2.0 ** -6
    off = w.detach().prod(1) * t["dy"].double().norm(dim=1) * size.sum(1)
    assert (t["dlogits"].double() - grads[0]).norm() <= 2.0 ** -6 * 2.0 ** 0.5 * off.norm()
    for name, grad in list(zip(v, grads))[1:]:
        assert relative(t["d" + name], grad) < 2.0 ** -5, name


SIZES = [(1, 4, 64, 32), (37, 8, 96, 72), (700, 40, 128, 64), (5000, 5, 60, 33)]


@pytest.mark.parametrize("tokens,experts,hidden,inner", SIZES)
def test_training_step(device, tokens, experts, hidden, inner):
    t, calls = training_step(tokens, experts, hidden, inner, tokens)
    calls.run()
    torch.cuda.synchronize()
    check_step(t)


@pytest.mark.parametrize("tokens,experts,hidden,inner", SIZES[1:])
def test_training_step_captured(device, tokens, experts, hidden, inner):
    """On a stream of its own and replayed from a graph, with new inputs and eager work between
    the replays; every replay gives the eager call's bits."""
    t, calls = training_step(tokens, experts, hidden, inner, tokens)
    other, eager = training_step(tokens, experts, hidden, inner, tokens)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        calls.run(torch.cuda.current_stream())
    outputs = ("ids", "weights", "offsets", "pos", "rows", "y", "dr", "dweights", "dlogits", "dx", "dw_gate", "dw_up", "dw_down")
    for seed in range(4):
        gen = torch.Generator(device="cuda:0")
        gen.manual_seed(seed)
        for name in ("logits", "x", "dy"):
            new = torch.randn(t[name].shape, device="cuda:0", generator=gen)
            t[name].copy_(new)
            other[name].copy_(new)
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        for name in outputs:
            assert torch.equal(t[name], other[name]), (seed, name)
    check_step(t)


def test_two_streams_at_once(device):
    """Two steps of different sizes whose calls alternate between two streams."""
    steps = [training_step(*size, seed=7) for size in SIZES[2:]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for (_, calls), stream in zip(steps, streams):
            calls.run(stream)
    torch.cuda.synchronize()
    for t, _ in steps:
        check_step(t)


def to_values(q, scale, hidden):
    """What quantised rows on the GPU stand for."""
    q, scale = q.cpu().numpy(), scale.cpu().numpy()
    code = np.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1)
    s = scale.transpose(1, 0, 2).reshape(q.shape[0], -1)[:, :q.shape[1] // 16]
    return values(code, s)[:, :hidden]


@pytest.mark.parametrize("tokens,top_k,experts,hidden,inner", [(1, 8, 16, 256, 96), (64, 2, 20, 320, 130), (600, 4, 6, 100, 72)])
def test_decode_in_4_bits(device, tokens, top_k, experts, hidden, inner):
    """Maps, rows quantised through them, two products with a quantisation between, and the
    combination: every operator on what the one before it wrote."""
    gen = np.random.default_rng(tokens)
    rows = tokens * top_k
    x = torch.randn(tokens, hidden, device="cuda:0").bfloat16()
    ids = torch.from_numpy(gen.integers(0, experts, (tokens, top_k), dtype=np.int32)).cuda()
    w = torch.rand(tokens, top_k, device="cuda:0")
    gate, up, down = (weights(gen, experts * n, k) for n, k in ((inner, hidden), (inner, hidden), (hidden, inner)))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    packed = {name: (dev(p), dev(layout(s - 5))) for name, (p, s, _) in (("gate", gate), ("up", up), ("down", down))}
    u8, i32 = dict(dtype=torch.uint8), dict(dtype=torch.int32)
    t = dict(offsets=zeros(experts + 1, **i32), pos=zeros(rows, **i32), route=zeros(rows, **i32))
    for name, k in (("x", hidden), ("a", inner)):
        blocks = -(-k // 32)
        t["q" + name], t["s" + name] = zeros(rows, 16 * blocks, **u8), zeros(-(-blocks // 8), rows, 8, **u8)
    t |= dict(a=zeros(rows, inner), r=zeros(rows, hidden, dtype=torch.float32), y=zeros(tokens, hidden, dtype=torch.float32))
    p = {name: v.data_ptr() for name, v in t.items()}
    calls = Calls()
    calls.add("sort_tokens", rr.SortTokensArgs(expert_ids=ids.data_ptr(), offsets=p["offsets"], route_pos=p["pos"],
                                               sorted_route=p["route"], tokens=tokens, experts=experts, top_k=top_k,
                                               hidden=hidden))
    calls.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=x.data_ptr(), sorted_route=p["route"], q=p["qx"],
                                                              scale=p["sx"], rows=rows, hidden=hidden, tokens=tokens,
                                                              top_k=top_k))
    common = dict(offsets=p["offsets"], rows=rows, experts=experts)
    calls.add("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
        q=p["qx"], q_scale=p["sx"], w=packed["gate"][0].data_ptr(), w_scale=packed["gate"][1].data_ptr(),
        w_up=packed["up"][0].data_ptr(), w_up_scale=packed["up"][1].data_ptr(), y=p["a"], hidden=hidden, output=inner, **common))
    calls.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=p["a"], q=p["qa"], scale=p["sa"], rows=rows, hidden=inner))
    calls.add("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
        q=p["qa"], q_scale=p["sa"], w=packed["down"][0].data_ptr(), w_scale=packed["down"][1].data_ptr(), y=p["r"],
        hidden=inner, output=hidden, dtype=CODES["f32"], **common))
    calls.add("combine_tokens", rr.CombineTokensArgs(y_sorted=p["r"], route_pos=p["pos"], route_weights=w.data_ptr(),
                                                     y=p["y"], tokens=tokens, top_k=top_k, hidden=hidden, dtype=CODES["f32"]))
    calls.run()
    torch.cuda.synchronize()

    offsets, pos, route = maps(ids.cpu(), experts)
    assert torch.equal(t["pos"].cpu(), pos) and torch.equal(t["offsets"].cpu(), offsets)
    source = x.double().cpu().numpy()[route.numpy() // top_k]
    code, scale = encode(source)
    xv = to_values(t["qx"], t["sx"], hidden)
    assert np.array_equal(xv, values(code, scale)[:, :hidden])
    av = to_values(t["qa"], t["sa"], inner)
    assert np.array_equal(av, values(*encode(t["a"].double().cpu().numpy()))[:, :inner])
    gv, uv, dv = (v[2].reshape(experts, -1, v[2].shape[1]) / 32 for v in (gate, up, down))
    a, size, r, r_size = (np.zeros((rows, n)) for n in (inner, inner, hidden, hidden))
    for e in range(experts):
        seg = slice(int(offsets[e]), int(offsets[e + 1]))
        g, u = xv[seg] @ gv[e][:, :hidden].T, xv[seg] @ uv[e][:, :hidden].T
        a[seg] = g / (1 + np.exp(-g)) * u
        g_err, u_err = (hidden * 2.0 ** -24 * (np.abs(xv[seg]) @ np.abs(m[e][:, :hidden]).T) for m in (gv, uv))
        size[seg] = 1.2 * (g_err + np.abs(g) * 2.0 ** -22) * (np.abs(u) + u_err) + (np.abs(g) + g_err) * u_err
        r[seg] = av[seg] @ dv[e][:, :inner].T
        r_size[seg] = inner * 2.0 ** -24 * (np.abs(av[seg]) @ np.abs(dv[e][:, :inner]).T)
    dbl = lambda v: torch.from_numpy(v)  # noqa: E731
    assert_within(t["a"].cpu(), dbl(a), dbl((np.abs(a) * 2.0 ** -20 + size) * (1 + 2.0 ** -8) + np.abs(a) * 2.0 ** -8 + 2.0 ** -130), "a")
    assert_within(t["r"].cpu(), dbl(r), dbl(r_size + np.abs(r) * 2.0 ** -24 + 2.0 ** -140), "r")
    terms = t["r"].double().cpu()[pos.view(tokens, top_k).long()] * w.double().cpu()[:, :, None]
    bound = (top_k + 1) * 2.0 ** -24 * terms.abs().sum(1) * 1.01
    assert_within(t["y"].cpu(), terms.sum(1), bound + 2.0 ** -140, "y")


@pytest.mark.parametrize("family", ["auto", "naive"])
@pytest.mark.parametrize("unit", [1, 9, 40, 300])
@pytest.mark.parametrize("name", list(OFFSETS))
def test_offsets_that_do_not_rise(device, name, unit, family):
    """Bounds are cut to [0, rows], one that falls counts as the largest before it, rows of none are
    left alone (few rows, short tiles, tiles of 128 and of 256 rows)."""
    rows, k, n = 10 * unit, 300, 40
    offsets = [unit * o for o in OFFSETS[name]]
    experts = len(offsets) - 1
    gen = np.random.default_rng(unit)
    q, qs, qv = weights(gen, rows, k)
    w, ws, wv = weights(gen, experts * n, k)
    import test_gpu_mxfp4 as t
    keep = t.offsets_of
    try:
        t.offsets_of = lambda counts: (torch.tensor(offsets, dtype=torch.int32, device="cuda:0"), rows)
        y = product(q, qs, [w], [ws], [0] * experts, k, n, "f32", "silu", family).t
    finally:
        t.offsets_of = keep
    at = bounds(offsets, rows)
    qv, wv = torch.from_numpy(qv).cuda(), torch.from_numpy(wv).cuda().view(experts, n, -1)
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda:0")
    for e in range(experts):
        seg = slice(at[e], at[e + 1])
        inside[seg] = True
        bound = k * 2.0 ** -24 * (qv[seg].abs() @ wv[e].abs().t().contiguous())
        want = qv[seg] @ wv[e].t().contiguous()
        assert_within(y[seg], want, bound + want.abs() * 2.0 ** -24 + 2.0 ** -140, f"expert {e}")
    assert (y[~inside].contiguous().view(torch.uint8) == 0xA5).all()


@pytest.mark.parametrize("counts,k,n,gated", [([3000, 0, 17], 96, 5000, False), ([40] * 500 + [0] * 500, 64, 70, True),
                                              ([200] * 700, 40, 33, False), ([9000], 520, 300, True),
                                              ([1, 0] * 512, 72, 130, False), ([6000] + [0] * 1023, 48, 20, False)])
def test_more_tiles_than_workgroups(device, counts, k, n, gated):
    """Several rounds of tiles, many experts (more than three stages of LDS leave bounds for), and
    rows that all go to one of them."""
    gen = np.random.default_rng(n)
    rows, e = sum(counts), len(counts)
    q, qs, qv = weights(gen, rows, k)
    parts = [weights(gen, e * n, k) for _ in range(1 + gated)]
    parts = [(p, s - 5, v / 32) for p, s, v in parts]
    y = product(q, qs, [p[0] for p in parts], [p[1] for p in parts], counts, k, n, "f32", "silu", "auto").t
    qv = torch.from_numpy(qv).cuda()
    wv = [torch.from_numpy(p[2]).cuda().view(e, n, -1) for p in parts]
    start = 0
    for x, c in enumerate(counts):
        if not c:
            continue
        seg = slice(start, start + c)
        start += c
        p = [qv[seg] @ w[x].t().contiguous() for w in wv]
        err = [k * 2.0 ** -24 * (qv[seg].abs() @ w[x].abs().t().contiguous()) for w in wv]
        want, bound = p[0], err[0]
        if gated:
            a = torch.nn.functional.silu(p[0])
            want = a * p[1]
            bound = (want.abs() * (2.0 ** -20 + 2.0 ** -22) + 1.2 * (err[0] + p[0].abs() * 2.0 ** -22) * (p[1].abs() + err[1])
                     + (a.abs() + 1.2 * err[0]) * err[1])
        assert_within(y[seg], want, bound + want.abs() * 2.0 ** -24 + 2.0 ** -140, f"expert {x}")


def test_rows_past_32_bits(device):
    """Sorted rows of 4.8 GB: copied, summed with their gradients, and quantised through the map."""
    tokens, top_k, hidden, experts = 300000, 4, 2000, 3
    x = torch.randn(tokens, hidden, device="cuda:0", dtype=torch.bfloat16)
    ids = torch.randint(0, experts, (tokens, top_k), device="cuda:0", dtype=torch.int32)
    rows = tokens * top_k
    t = dict(offsets=zeros(experts + 1, dtype=torch.int32), pos=zeros(rows, dtype=torch.int32),
             route=zeros(rows, dtype=torch.int32), out=torch.empty(rows, hidden, dtype=torch.bfloat16, device="cuda:0"),
             y=zeros(tokens, hidden), dw=zeros(rows, dtype=torch.float32))
    p = {name: v.data_ptr() for name, v in t.items()}
    calls = Calls()
    calls.add("sort_tokens", rr.SortTokensArgs(x=x.data_ptr(), expert_ids=ids.data_ptr(), offsets=p["offsets"],
                                               route_pos=p["pos"], sorted_route=p["route"], x_sorted=p["out"], tokens=tokens,
                                               experts=experts, top_k=top_k, hidden=hidden))
    calls.add("sort_tokens_backward", rr.SortTokensBackwardArgs(dx_sorted=p["out"], route_pos=p["pos"], dx=p["y"],
                                                                tokens=tokens, top_k=top_k, hidden=hidden))
    calls.run()
    key = ids.reshape(-1).long()
    order = torch.sort(key, stable=True).indices
    assert torch.equal(t["route"].long(), order)
    for part in torch.arange(rows, device="cuda:0").split(100000):
        assert torch.equal(t["out"][part], x[order[part] // top_k])
    assert torch.equal(t["y"], 4 * x)  # (four times a number is exact)
    back = Calls()
    back.add("combine_tokens_backward", rr.CombineTokensBackwardArgs(
        dy=x.data_ptr(), y_sorted=p["out"], route_pos=p["pos"], dy_sorted=p["out"], droute_weights=p["dw"], tokens=tokens,
        top_k=top_k, hidden=hidden))
    back.run()
    for part in torch.arange(rows, device="cuda:0").split(100000):
        assert torch.equal(t["out"][part], x[order[part] // top_k])
    want = torch.cat([v.double().square().sum(1) for v in x.split(50000)])
    assert_within(t["dw"].view(tokens, top_k), want[:, None].expand(-1, top_k),
                  ((hidden + 1) * 2.0 ** -24 * want)[:, None].expand(-1, top_k), "dw")
    blocks = -(-hidden // 32)
    q, s = zeros(rows, 16 * blocks, dtype=torch.uint8), zeros(-(-blocks // 8), rows, 8, dtype=torch.uint8)
    quant = Calls()
    quant.add("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=x.data_ptr(), sorted_route=p["route"], q=q.data_ptr(),
                                                              scale=s.data_ptr(), rows=rows, hidden=hidden, tokens=tokens,
                                                              top_k=top_k))
    quant.run()
    for part in (torch.arange(64), torch.arange(rows - 64, rows)):
        code, scale = encode(x[order[part.cuda()] // top_k].double().cpu().numpy())
        got = to_values(q[part.cuda()], s[:, part.cuda()], hidden)
        assert np.array_equal(got, values(code, scale)[:, :hidden])


@pytest.mark.parametrize("rows,experts,n,k,gated", [(40, 33, 16384, 16384, False), (2600, 20, 16384, 16384, False),
                                                    (300000, 2, 33, 16384, False)])
def test_products_past_32_bits(device, rows, experts, n, k, gated):
    """Weights of 4.4 and 2.7 GB (few rows, tiles), rows of 2.5 GB: the last expert's results."""
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(k)
    counts = [0] * experts
    counts[0], counts[-1] = rows // 2, rows - rows // 2
    blocks, slices = k // 32, k // 256

    def random(*shape):
        return torch.randint(0, 256, shape, device="cuda:0", generator=gen, dtype=torch.uint8)

    q, w = random(rows, 16 * blocks), random(experts, n, 16 * blocks)
    qs = torch.randint(120, 123, (slices, rows, 8), device="cuda:0", generator=gen, dtype=torch.uint8)
    ws = torch.randint(120, 123, (slices, experts * n, 8), device="cuda:0", generator=gen, dtype=torch.uint8)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda:0")
    y = Buf(shape=(rows, n), dtype=torch.float32)
    calls = Calls()
    calls.add("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
        q=q.data_ptr(), q_scale=qs.data_ptr(), w=w.data_ptr(), w_scale=ws.data_ptr(), offsets=offsets.data_ptr(), y=y.ptr,
        rows=rows, experts=experts, hidden=k, output=n, dtype=CODES["f32"]))
    calls.run()
    assert y.intact()
    last, channels = torch.arange(rows - 20, rows, device="cuda:0"), torch.arange(n - 30, n, device="cuda:0")
    qv = torch.from_numpy(to_values(q[last], qs[:, last], k)).cuda()
    wv = torch.from_numpy(to_values(w[-1][channels], ws[:, (experts - 1) * n + channels], k)).cuda()
    got = y.t[last][:, channels]
    want = qv @ wv.t().contiguous()
    assert_within(got, want, k * 2.0 ** -24 * (qv.abs() @ wv.abs().t().contiguous()), "last rows and channels")
