"""The operators that take tokens to their experts and back, with their gradients,
and the experts' products in microscaled 4-bit floating point.

A case is a dict of plain values. "op" says what one pass computes:

  sort     sort_tokens: the routes of all tokens in order of their experts and
           the tokens' rows in that order; with train also sort_tokens_backward,
           the sum of a token's rows' gradients;
  combine  combine_tokens: the sum of a token's rows with its routes' weights;
           with train also combine_tokens_backward (gradients of the rows and of
           the weights) and topk_gate_backward (of the router's logits);
  fp4      quantize_rows_mxfp4 of the routed rows, then mxfp4_grouped_gemm
           (gated: two weights, the activation and the product of the two in it).
           Blocks of 32 elements share a power of two.

`own = False` computes a pass in plain torch: float32 whatever the inputs'
type, rounded once at the end.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]  # the magnitudes of four bits


def listed() -> list[dict]:
    return [
        # Decoding one token of a fine-grained model: eight of 128 experts; latency.
        dict(name="sort_token", op="sort", dtype="bf16", x_dtype="bf16", tokens=1, top_k=8, experts=128, hidden=2048,
             skew=0.0, masked=0.0, train=False),
        # A padded batch of odd rows over nine experts, FP32 rows of the norm cast where they enter the experts.
        dict(name="sort_ragged", op="sort", dtype="f16", x_dtype="f32", tokens=3001, top_k=2, experts=9, hidden=1023,
             skew=0.6, masked=0.2, train=False),
        # A prefill of a wide layer, top-2 of eight.
        dict(name="sort_prefill", op="sort", dtype="bf16", x_dtype="bf16", tokens=16384, top_k=2, experts=8,
             hidden=4096, skew=0.6, masked=0.0, train=False),
        # A training step of a fine-grained layer, with the rows' gradients summed.
        dict(name="sort_train", op="sort", dtype="bf16", x_dtype="bf16", tokens=8192, top_k=8, experts=128,
             hidden=2048, skew=0.6, masked=0.0, train=True),
        # A decode batch of 64 tokens: latency.
        dict(name="combine_decode", op="combine", dtype="bf16", y_dtype="bf16", tokens=64, top_k=8, experts=128,
             hidden=2048, skew=0.5, masked=0.0, train=False),
        # A training step over odd rows with padding tokens, a few experts.
        dict(name="combine_ragged", op="combine", dtype="f16", y_dtype="f16", tokens=3001, top_k=2, experts=9,
             hidden=1023, skew=0.6, masked=0.2, train=True),
        # A prefill of a wide layer; the block's result is FP32, as the norm after it takes it.
        dict(name="combine_prefill", op="combine", dtype="bf16", y_dtype="f32", tokens=16384, top_k=2, experts=8,
             hidden=4096, skew=0.6, masked=0.0, train=False),
        # A training step of a fine-grained layer, with the gradients of rows, weights and logits.
        dict(name="combine_train", op="combine", dtype="bf16", y_dtype="bf16", tokens=8192, top_k=8, experts=128,
             hidden=2048, skew=0.6, masked=0.0, train=True),
        # Decoding one token of a wide model: two of eight experts with one row each, all of it weight traffic.
        dict(name="fp4_token", op="fp4", dtype="bf16", tokens=1, top_k=2, experts=8, hidden=4096, output=14336,
             skew=0.0, gated=True, act="silu"),
        # The first expert product of a decode batch over many fine-grained experts.
        dict(name="fp4_decode", op="fp4", dtype="bf16", tokens=64, top_k=2, experts=128, hidden=2048, output=768,
             skew=0.5, gated=True, act="silu"),
        # Widths that nothing was rounded for, the other activation and type.
        dict(name="fp4_ragged", op="fp4", dtype="f16", tokens=3001, top_k=2, experts=9, hidden=1023, output=1535,
             skew=0.6, gated=True, act="gelu"),
        # An expert product of a wide layer in prefill.
        dict(name="fp4_prefill", op="fp4", dtype="bf16", tokens=8192, top_k=2, experts=8, hidden=4096, output=14336,
             skew=0.6, gated=False, act="silu"),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo: int, hi: int, odd: bool) -> int:
    """A row width: any number, or (most models) a multiple of 32."""
    n = _log_uniform(rng, lo, hi)
    return n if odd else max(lo, n // 32 * 32)


def draw(rng) -> dict:
    op = rng.choice(["sort", "combine", "fp4", "fp4"])
    odd = rng.random() < 0.4
    experts = _log_uniform(rng, 1, 256)
    top_k = rng.randint(1, min(8, experts))
    skew = rng.choice([0.0, 0.6, 1.0])
    if op != "fp4":
        dtype = rng.choice(["bf16", "f16", "f32"])
        other = rng.choice([dtype, dtype, "f32"])
        # no more rows than the widest listed step has
        most = 8192 * 8 * 2048 // (2 if "f32" in (dtype, other) else 1)
        hidden = _width(rng, 64, 8192, odd)
        tokens = _log_uniform(rng, 1, min(16384, most // (hidden * top_k)))
        return {"op": op, "dtype": dtype, ("x_dtype" if op == "sort" else "y_dtype"): other, "tokens": tokens,
                "top_k": top_k, "experts": experts, "hidden": hidden, "skew": skew,
                "masked": rng.choice([0.0, 0.0, 0.2]), "train": rng.random() < 0.5}
    hidden = _width(rng, 64, 4096, odd)
    # the weights no larger than the widest listed layer's
    output = _width(rng, 64, min(14336, 8 * 4096 * 14336 // (experts * hidden)), odd)
    gated = rng.random() < 0.5
    return dict(op=op, dtype=rng.choice(["bf16", "f16"]), tokens=_log_uniform(rng, 1, 16384 // (top_k * (1 + gated))),
                top_k=top_k, experts=experts, hidden=hidden, output=output, skew=skew, gated=gated,
                act=rng.choice(["silu", "gelu"]))


# ---- inputs ----

def _gen(seed: int):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, device=DEVICE, generator=gen).mul_(std).to(dtype)


def _routes(case: dict, gen):
    """Distinct experts of every token by a Zipf(skew) popularity in random order of the
    experts, weights of the softmax over their logits, ids -1 for the padding tokens."""
    t, e = case["tokens"], case["experts"]
    popularity = -case["skew"] * torch.log1p(torch.randperm(e, device=DEVICE, generator=gen).float())
    gumbel = -torch.log(-torch.log(torch.rand(t, e, device=DEVICE, generator=gen).clamp_(1e-7, 1.0 - 1e-6)))
    logits, ids = (popularity + gumbel).topk(case["top_k"], dim=1)
    if case.get("masked"):
        ids[torch.rand(t, device=DEVICE, generator=gen) < case["masked"]] = -1
    return ids.to(torch.int32).contiguous(), torch.softmax(logits, dim=1).contiguous()


def _maps(ids, experts: int):
    """offsets, route_pos and sorted_route of the routes' stable order."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    offsets = torch.zeros(experts + 2, dtype=torch.int64, device=DEVICE)
    offsets[1:] = torch.bincount(key, minlength=experts + 1).cumsum(0)
    rank = torch.arange(flat.numel(), device=DEVICE)
    placed = rank < offsets[experts]
    position = torch.empty_like(order)
    position[order] = torch.where(placed, rank, torch.full_like(rank, -1))
    route = torch.where(placed, order, torch.full_like(order, -1))
    return offsets[:experts + 1].int(), position.int(), route.int()


def _inputs(case: dict, seed: int) -> dict:
    gen = _gen(seed)
    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    dtype = TYPES[case["dtype"]]
    ids, weights = _routes(case, gen)
    if case["op"] == "sort":
        inp = {"ids": ids, "x": _normal(gen, t, h, dtype=TYPES[case["x_dtype"]])}
        if case["train"]:
            inp["dx_sorted"] = _normal(gen, t * k, h, dtype=dtype)
        return inp
    offsets, position, route = _maps(ids, case["experts"])
    if case["op"] == "combine":
        inp = {"ids": ids, "weights": weights, "position": position, "y_sorted": _normal(gen, t * k, h, dtype=dtype)}
        if case["train"]:
            inp["dy"] = _normal(gen, t, h, dtype=TYPES[case["y_dtype"]])
        return inp
    # activations of uneven channels with a few large ones, as they come out of a norm
    channel = torch.exp(_normal(gen, h, std=0.5))
    channel[torch.rand(h, device=DEVICE, generator=gen) < 0.01] *= 8.0
    inp = {"x": (_normal(gen, t, h) * channel).to(dtype), "offsets": offsets, "route": route}
    e, n, blocks = case["experts"], case["output"], (h + 31) // 32
    for name in ["w", "w_up"] if case["gated"] else ["w"]:
        q = torch.randint(0, 256, (e, n, 16 * blocks), device=DEVICE, generator=gen, dtype=torch.uint8)
        if h % 32:  # elements past the row are zeros
            first = torch.arange(0, 32 * blocks, 2, device=DEVICE)
            q &= torch.where(first + 1 < h, 255, torch.where(first < h, 15, 0)).to(torch.uint8)
        inp[name] = q
        # powers of two about a channel's largest weight, uneven over the blocks
        base = 125 - int(round(0.5 * math.log2(h)))
        inp[name + "_scale"] = torch.randint(base - 1, base + 2, (e, n, blocks), device=DEVICE, generator=gen,
                                             dtype=torch.uint8)
    return inp


def prepare(case: dict, seed: int) -> dict:
    inp = _inputs(case, seed)
    state = {"case": case, "inputs": inp, "own": own}
    if own:
        _plan(state)
    return state


# ---- the framework's operators ----

def _plan(state: dict) -> None:
    import raggedroute_amd as rr

    case, inp = state["case"], state["inputs"]
    codes = {"f32": int(rr.ScalarType.kFp32), "f16": int(rr.ScalarType.kFp16), "bf16": int(rr.ScalarType.kBf16)}
    dtype, code = TYPES[case["dtype"]], codes[case["dtype"]]
    stream = torch.cuda.current_stream().cuda_stream
    keep = state["buffers"] = {}
    calls = state["calls"] = []
    p = {name: value.data_ptr() for name, value in inp.items()}

    def new(name, *shape, dtype=dtype):
        # (rows that no route leads to stay as they are: zeros)
        keep[name] = torch.zeros(*shape, dtype=dtype, device=DEVICE)
        return keep[name].data_ptr()

    def call(entry, args, workspace_size):
        size = workspace_size(args)
        workspace = torch.empty(size, dtype=torch.uint8, device=DEVICE) if size else None
        keep["workspace%d" % len(calls)] = workspace
        calls.append((entry, args, rr.RuntimeContext(stream=stream, workspace_bytes=size,
                                                     workspace=workspace.data_ptr() if size else None)))

    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    rows = t * k
    if case["op"] == "sort":
        x_type, x_code = TYPES[case["x_dtype"]], codes[case["x_dtype"]]
        position = new("position", rows, dtype=torch.int32)
        call(rr.sort_tokens,
             rr.SortTokensArgs(x=p["x"], expert_ids=p["ids"], route_pos=position,
                               offsets=new("offsets", case["experts"] + 1, dtype=torch.int32),
                               sorted_route=new("route", rows, dtype=torch.int32), x_sorted=new("x_sorted", rows, h),
                               tokens=t, experts=case["experts"], top_k=k, hidden=h, dtype=code, x_dtype=x_code),
             rr.get_sort_tokens_workspace_size)
        outputs = ["offsets", "position", "route", "x_sorted"]
        if case["train"]:
            call(rr.sort_tokens_backward,
                 rr.SortTokensBackwardArgs(dx_sorted=p["dx_sorted"], route_pos=position, dx=new("dx", t, h, dtype=x_type),
                                           tokens=t, top_k=k, hidden=h, dtype=code, x_dtype=x_code),
                 rr.get_sort_tokens_backward_workspace_size)
            outputs.append("dx")
    elif case["op"] == "combine":
        y_type, y_code = TYPES[case["y_dtype"]], codes[case["y_dtype"]]
        common = dict(y_sorted=p["y_sorted"], route_pos=p["position"], route_weights=p["weights"], tokens=t, top_k=k,
                      hidden=h, dtype=code, y_dtype=y_code)
        call(rr.combine_tokens, rr.CombineTokensArgs(y=new("y", t, h, dtype=y_type), **common),
             rr.get_combine_tokens_workspace_size)
        outputs = ["y"]
        if case["train"]:
            dw = new("dweights", t, k, dtype=torch.float32)
            call(rr.combine_tokens_backward,
                 rr.CombineTokensBackwardArgs(dy=p["dy"], dy_sorted=new("dy_sorted", rows, h), droute_weights=dw, **common),
                 rr.get_combine_tokens_backward_workspace_size)
            call(rr.topk_gate_backward,
                 rr.TopKGateBackwardArgs(expert_ids=p["ids"], weights=p["weights"], dweights=dw,
                                         dlogits=new("dlogits", t, case["experts"], dtype=torch.float32), tokens=t,
                                         experts=case["experts"], top_k=k), rr.get_topk_gate_backward_workspace_size)
            outputs += ["dy_sorted", "dweights", "dlogits"]
    else:
        e, n, blocks = case["experts"], case["output"], (h + 31) // 32
        slices = (blocks + 7) // 8
        q, s = new("q", rows, 16 * blocks, dtype=torch.uint8), new("q_scale", slices, rows, 8, dtype=torch.uint8)
        call(rr.quantize_rows_mxfp4,
             rr.QuantizeRowsMxfp4Args(x=p["x"], sorted_route=p["route"], q=q, scale=s, rows=rows, hidden=h, tokens=t,
                                      top_k=k, dtype=code), rr.get_quantize_rows_mxfp4_workspace_size)
        weights = {}
        for name in ["w", "w_up"] if case["gated"] else ["w"]:
            # the scales of eight blocks side by side for every row, laid out once
            scale = torch.zeros(e * n, 8 * slices, dtype=torch.uint8, device=DEVICE)
            scale[:, :blocks] = inp[name + "_scale"].view(e * n, blocks)
            keep[name + "_scale"] = scale.view(e * n, slices, 8).transpose(0, 1).contiguous()
            weights.update({name: p[name], name + "_scale": keep[name + "_scale"].data_ptr()})
        act = int({"silu": rr.Activation.kSilu, "gelu": rr.Activation.kGeluTanh}[case["act"]])
        call(rr.mxfp4_grouped_gemm,
             rr.Mxfp4GroupedGemmArgs(q=q, q_scale=s, offsets=p["offsets"], y=new("y", rows, n), rows=rows, experts=e,
                                     hidden=h, output=n, activation=act, dtype=code, **weights),
             rr.get_mxfp4_grouped_gemm_workspace_size)
        outputs = ["y"]
    state["outputs"] = {name: keep[name] for name in outputs}


# ---- the plain forms ----

def _plain_sort(case: dict, inp: dict) -> dict:
    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    dtype = TYPES[case["dtype"]]
    offsets, position, route = _maps(inp["ids"], case["experts"])
    token = (route.clamp(min=0) // k).long()
    rows = inp["x"][token].to(dtype)
    out = {"offsets": offsets, "position": position, "route": route,
           "x_sorted": torch.where((route >= 0)[:, None], rows, torch.zeros_like(rows))}
    if case["train"]:
        placed = (position >= 0)[:, None]
        back = torch.where(placed, inp["dx_sorted"][position.clamp(min=0).long()].float(), torch.zeros((), device=DEVICE))
        out["dx"] = back.view(t, k, h).sum(1).to(inp["x"].dtype)
    return out


def _plain_combine(case: dict, inp: dict) -> dict:
    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    dtype, y_type = TYPES[case["dtype"]], TYPES[case["y_dtype"]]
    position, w = inp["position"].view(t, k), inp["weights"]
    placed = position >= 0
    rows = inp["y_sorted"][position.clamp(min=0).long()].float() * placed[:, :, None]
    out = {"y": (rows * w[:, :, None]).sum(1).to(y_type)}
    if case["train"]:
        dy = inp["dy"].float()
        out["dy_sorted"] = torch.zeros(t * k, h, dtype=dtype, device=DEVICE)
        back = (dy[:, None, :] * w[:, :, None]).to(dtype)
        out["dy_sorted"][position[placed].long()] = back[placed]
        dw = (rows * dy[:, None, :]).sum(2)
        out["dweights"] = dw
        # (differences of nearby numbers)
        w64, dw64 = w.double(), dw.double()
        grad = (w64[:, :, None] * w64[:, None, :] * (dw64[:, :, None] - dw64[:, None, :])).sum(2).float()
        valid = inp["ids"] >= 0
        dlogits = torch.zeros(t, case["experts"], device=DEVICE)
        out["dlogits"] = dlogits.scatter_add_(1, inp["ids"].clamp(min=0).long(), grad * valid)
    return out


def _to_fp4(x):
    """Rows of float32 as the values that their 4-bit elements and blocks' powers of two stand for."""
    rows, h = x.shape
    pad = -h % 32
    blocks = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, 32)
    power = (torch.frexp(blocks.abs().amax(2, keepdim=True)).exponent - 3).clamp(min=-127)
    v = torch.ldexp(blocks, -power)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    return torch.ldexp(torch.copysign(a, v), power).view(rows, -1)[:, :h]


def _fp4_values(q, scale, h: int):
    """Packed weights as float32."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], device=DEVICE)
    v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], dim=-1).view(*q.shape[:-1], -1, 32)
    return torch.ldexp(v, scale.int()[..., None] - 127).view(*q.shape[:-1], -1)[..., :h]


def _activation(name: str, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_fp4(case: dict, inp: dict) -> dict:
    h = case["hidden"]
    x = _to_fp4(inp["x"].float())[(inp["route"] // case["top_k"]).long()]
    bounds = inp["offsets"].tolist()
    y = torch.zeros(x.shape[0], case["output"], dtype=inp["x"].dtype, device=DEVICE)
    for e in range(case["experts"]):
        rows = slice(bounds[e], bounds[e + 1])
        if rows.start == rows.stop:
            continue
        p = [x[rows] @ _fp4_values(inp[name][e], inp[name + "_scale"][e], h).t()
             for name in (("w", "w_up") if case["gated"] else ("w",))]
        y[rows] = (_activation(case["act"], p[0]) * p[1] if case["gated"] else p[0]).to(y.dtype)
    return {"y": y}


_PLAIN = {"sort": _plain_sort, "combine": _plain_combine, "fp4": _plain_fp4}


def run(state: dict) -> dict:
    if not state["own"]:
        return _PLAIN[state["case"]["op"]](state["case"], state["inputs"])
    for entry, args, context in state["calls"]:
        status = entry(args, context)
        if not status.ok():
            raise RuntimeError(status.message)
    return state["outputs"]


def work(case: dict) -> dict:
    """Each input read once and each output written once (weights of experts that can have
    rows, placed rows), and the products' multiply-adds."""
    t, k, h, e = case["tokens"], case["top_k"], case["hidden"], case["experts"]
    size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    placed = (1.0 - case.get("masked", 0.0)) * t * k
    if case["op"] == "sort":
        x_size = torch.empty(0, dtype=TYPES[case["x_dtype"]]).element_size()
        moved, flops = x_size * t * h + size * placed * h + 12 * t * k + 4 * (e + 1), 0
        if case["train"]:
            moved += size * placed * h + x_size * t * h
            flops = placed * h
        return {"bytes": int(moved), "flops": int(flops)}
    if case["op"] == "combine":
        y_size = torch.empty(0, dtype=TYPES[case["y_dtype"]]).element_size()
        moved, flops = size * placed * h + y_size * t * h + 8 * t * k, 2 * placed * h
        if case["train"]:
            # dy, dy_sorted, the weights' gradients, the ids and the logits' gradients
            moved += y_size * t * h + size * placed * h + 8 * t * k + 4 * t * e
            flops += 3 * placed * h + 4 * t * k * k
        return {"bytes": int(moved), "flops": int(flops)}
    n, weights = case["output"], 2 if case["gated"] else 1
    blocks = (h + 31) // 32
    moved = size * t * h + 4 * t * k + 4 * (e + 1) + min(e, t * k) * weights * n * 17 * blocks + size * t * k * n
    return {"bytes": int(moved), "flops": int(2 * weights * t * k * h * n)}


# ---- results in 64 bits ----

def exact(case: dict, seed: int):
    inp = _inputs(case, seed)
    return {"sort": _exact_sort, "combine": _exact_combine, "fp4": _exact_fp4}[case["op"]](case, inp)


def _exact_sort(case: dict, inp: dict) -> dict:
    """By counting over the experts on the host."""
    ids = inp["ids"].reshape(-1).cpu().numpy()
    k, e = case["top_k"], case["experts"]
    order = np.concatenate([np.flatnonzero(ids == x) for x in range(e)])
    counts = np.array([(ids == x).sum() for x in range(e)])
    position, route = np.full(ids.size, -1, np.int32), np.full(ids.size, -1, np.int32)
    position[order] = np.arange(order.size)
    route[:order.size] = order
    rows = torch.zeros(ids.size, case["hidden"], dtype=torch.float64, device=DEVICE)
    token = torch.from_numpy(order // k).to(DEVICE)
    rows[:order.size] = inp["x"].double()[token]
    out = {"offsets": torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).to(DEVICE),
           "position": torch.from_numpy(position).to(DEVICE), "route": torch.from_numpy(route).to(DEVICE), "x_sorted": rows}
    if case["train"]:
        dx = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=DEVICE)
        out["dx"] = dx.index_add_(0, token, inp["dx_sorted"][:order.size].double())
    return out


def _exact_combine(case: dict, inp: dict) -> dict:
    """By differentiating the operator's formula in float64, rank by rank; the logits'
    gradient by differentiating the softmax over logits whose softmax the weights are."""
    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    train = case["train"]
    rows = inp["y_sorted"].double().requires_grad_(train)
    w = inp["weights"].double().requires_grad_(train)
    y = torch.zeros(t, h, dtype=torch.float64, device=DEVICE)
    position = inp["position"].view(t, k).long()
    for j in range(k):
        token = torch.nonzero(position[:, j] >= 0).squeeze(1)
        y = y.index_add(0, token, w[token, j, None] * rows[position[token, j]])
    out = {"y": y.detach()}
    if train:
        out["dy_sorted"], out["dweights"] = torch.autograd.grad(y, (rows, w), inp["dy"].double())
        ids = inp["ids"].long()
        logits = torch.zeros(t, case["experts"], dtype=torch.float64, device=DEVICE)
        logits.scatter_(1, ids.clamp(min=0), torch.log(w.detach()))
        logits.requires_grad_(True)
        chosen = torch.softmax(logits.gather(1, ids.clamp(min=0)), dim=1) * (ids >= 0)
        out["dlogits"] = torch.autograd.grad(chosen, logits, out["dweights"])[0]
    return out


def _exact_fp4(case: dict, inp: dict) -> dict:
    """The rows' elements by their distances from the fifteen values, ties to the even code."""
    h = case["hidden"]
    x = inp["x"].double()
    x = torch.nn.functional.pad(x, (0, -h % 32)).view(x.shape[0], -1, 32)
    top = x.abs().amax(2, keepdim=True)
    power = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=1e-300))) - 2, torch.full_like(top, -127)).clamp(min=-127)
    v = (x.abs() / torch.exp2(power)).clamp(max=6.0)
    code = torch.zeros(v.shape, dtype=torch.int64, device=DEVICE)
    for c in range(7):
        middle = (E2M1[c] + E2M1[c + 1]) / 2
        # (a tie at an even code stays there, at an odd one goes on)
        code += (v > middle) if c % 2 == 0 else (v >= middle)
    table = torch.tensor(E2M1, dtype=torch.float64, device=DEVICE)
    x = (torch.sign(x) * table[code] * torch.exp2(power)).view(x.shape[0], -1)
    signed = torch.cat([table, -table])
    y = torch.zeros(inp["route"].numel(), case["output"], dtype=torch.float64, device=DEVICE)
    offsets = inp["offsets"].cpu().numpy()
    for e in range(case["experts"]):
        first, last = int(offsets[e]), int(offsets[e + 1])
        if first == last:
            continue
        a = x[(inp["route"][first:last] // case["top_k"]).long()]
        parts = []
        for name in ("w", "w_up") if case["gated"] else ("w",):
            q = inp[name][e]
            w = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=DEVICE)
            w[:, 0::2], w[:, 1::2] = signed[(q & 15).long()], signed[(q >> 4).long()]
            w *= torch.exp2(inp[name + "_scale"][e].double() - 127).repeat_interleave(32, dim=1)
            parts.append(a @ w.t().contiguous())
        g = parts[0]
        if case["gated"]:
            t = g if case["act"] == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)
            g = g * torch.sigmoid(t) * parts[1]
        y[first:last] = g
    return {"y": y}
