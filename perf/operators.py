"""The operators of a mixture-of-experts block around the routing chain, as a
training or serving program calls them.

A case is a dict of plain values. "op" says what one pass computes:

  ffn    gated_ffn: g = x Wg, u = x Wu, a = act(g) u, y = a Wd over the routed
         rows of every expert; with train also gated_ffn_backward, which gives
         the gradients of x and of the three weights;
  norm   block_norm: h = x + scale gate N(y; w_post), n = N(h; w_pre), with
         N(v; w) = v / sqrt(mean(v^2) + eps) w; with train also
         block_norm_backward;
  int8   quantize_rows of the routed rows, then int8_grouped_gemm with a scale
         per row and per expert and output channel (gated: two weights, the
         activation and the product of the two in it).

`own = False` computes a pass in plain torch: float32 whatever the inputs'
type, rounded once at the end.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
SCALE = 0.5  # residual scale of the block_norm cases
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # Decoding one token of a wide model: two of eight experts with one row each, all of it weight traffic.
        dict(name="ffn_token", op="ffn", dtype="bf16", rows=2, experts=8, active=2, hidden=4096, inner=14336,
             skew=0.0, act="silu", train=False),
        # A decode step over narrow experts, a few rows each: launches and latency.
        dict(name="ffn_small", op="ffn", dtype="f16", rows=64, experts=64, active=40, hidden=256, inner=128,
             skew=0.0, act="silu", train=False),
        # A decode batch of 64 tokens over many fine-grained experts.
        dict(name="ffn_decode", op="ffn", dtype="bf16", rows=128, experts=128, active=80, hidden=2048, inner=768,
             skew=0.5, act="silu", train=False),
        # Widths that nothing was rounded for, an expert without rows, the other activation and type.
        dict(name="ffn_ragged", op="ffn", dtype="f16", rows=6002, experts=9, active=8, hidden=1023, inner=1535,
             skew=0.6, act="gelu", train=False),
        # Large-batch prefill of a fine-grained layer with skewed routing.
        dict(name="ffn_prefill", op="ffn", dtype="bf16", rows=32768, experts=128, active=128, hidden=2048, inner=768,
             skew=1.0, act="silu", train=False),
        # A training step of a mid-size layer.
        dict(name="ffn_train", op="ffn", dtype="bf16", rows=8192, experts=64, active=64, hidden=1024, inner=512,
             skew=0.6, act="silu", train=True),
        # A training step of a wide layer: the largest products.
        dict(name="ffn_train_wide", op="ffn", dtype="bf16", rows=8192, experts=8, active=8, hidden=4096, inner=14336,
             skew=0.6, act="silu", train=True),
        # The norms around the block for four decoded tokens, a gate for each.
        dict(name="norm_token", op="norm", dtype="bf16", tokens=4, hidden=4096, gate_tokens=1, post=True, train=False),
        # The norms of a prefill: eight sequences with a gate row for each.
        dict(name="norm_prefill", op="norm", dtype="bf16", tokens=16384, hidden=4096, gate_tokens=2048, post=True,
             train=False),
        # The norms of a training step, with every gradient.
        dict(name="norm_train", op="norm", dtype="bf16", tokens=8192, hidden=4096, gate_tokens=1024, post=True,
             train=True),
        # The first expert product of a quantised decode batch.
        dict(name="int8_decode", op="int8", dtype="bf16", rows=128, experts=128, active=80, hidden=2048, output=768,
             skew=0.5, gated=True),
        # A quantised expert product of a wide layer in prefill.
        dict(name="int8_prefill", op="int8", dtype="bf16", rows=16384, experts=8, active=8, hidden=4096, output=14336,
             skew=0.6, gated=False),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo: int, hi: int, odd: bool) -> int:
    """A row width: any number, or (most models) a multiple of 32."""
    n = _log_uniform(rng, lo, hi)
    n = n if odd else max(lo, n // 32 * 32)
    return n if n != 3072 else n - 32  # (no configuration here has that width)


def draw(rng) -> dict:
    op = rng.choice(["ffn", "ffn", "ffn", "norm", "int8", "int8"])
    odd = rng.random() < 0.4
    if op == "norm":
        tokens = _log_uniform(rng, 1, 16384)
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), tokens=tokens,
                    hidden=_width(rng, 64, 8192 if tokens < 8192 else 4096, odd),
                    gate_tokens=rng.choice([0, 1, _log_uniform(rng, 1, tokens)]), post=rng.random() < 0.7,
                    train=rng.random() < 0.5)
    experts = _log_uniform(rng, 1, 128)
    hidden = _width(rng, 64, 4096, odd)
    # the weights no larger than the widest listed layer's
    width = _width(rng, 64, min(14336, 8 * 4096 * 14336 // (experts * hidden)), odd)
    train = op == "ffn" and rng.random() < 0.4
    rows = _log_uniform(rng, 1, 8192 if train else 16384)
    case = dict(op=op, dtype=rng.choice(["bf16", "f16"]), rows=rows, experts=experts,
                active=max(1, min(rows, experts - rng.randrange(2))), hidden=hidden)
    if op == "ffn":
        return dict(case, inner=width, skew=rng.choice([0.0, 0.6, 1.0]), act=rng.choice(["silu", "gelu"]), train=train)
    return dict(case, output=width, skew=rng.choice([0.0, 0.6, 1.0]), gated=rng.random() < 0.5)


# ---- inputs ----

def _counts(case: dict, seed: int) -> list[int]:
    """Rows of every expert: `active` of them (at random) have one at least, the
    others follow a Zipf(skew) popularity."""
    rng = np.random.default_rng(seed)
    active = case["active"]
    p = (1.0 + np.arange(active)) ** -case["skew"]
    counts = np.zeros(case["experts"], dtype=np.int64)
    counts[rng.permutation(case["experts"])[:active]] = 1 + rng.multinomial(case["rows"] - active, p / p.sum())
    return counts.tolist()


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype):
        return torch.randn(*shape, device=DEVICE, generator=gen).mul_(std).add_(mean).to(dtype)

    k = case["hidden"]
    if case["op"] == "norm":
        t, every = case["tokens"], case["gate_tokens"]
        inp = {"x": normal(t, k, std=2.0), "y": normal(t, k), "w_pre": normal(k, std=0.2, mean=1.0)}
        if case["post"]:
            inp["w_post"] = normal(k, std=0.2, mean=1.0)
        if every:
            inp["gate"] = normal((t + every - 1) // every, k, std=0.5, mean=0.5)
        if case["train"]:
            inp["dh"], inp["dn"] = normal(t, k), normal(t, k)
        return inp
    counts = _counts(case, seed)
    r, e = case["rows"], case["experts"]
    inp = {"counts": counts,
           "offsets": torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEVICE),
           "x": normal(r, k)}
    if case["op"] == "ffn":
        f = case["inner"]
        inp["w_gate"] = normal(e, k, f, std=k ** -0.5)
        inp["w_up"] = normal(e, k, f, std=k ** -0.5)
        inp["w_down"] = normal(e, f, k, std=f ** -0.5)
        if case["train"]:
            inp["dy"] = normal(r, k)
        return inp
    n = case["output"]
    for name in ["w_gate", "w_up"] if case["gated"] else ["w"]:
        inp[name] = torch.randint(-127, 128, (e, n, k), device=DEVICE, generator=gen, dtype=torch.int8)
        # a channel's scale: its largest weight (about 4 of k^-0.5) over 127, uneven over the channels
        inp[name + "_scale"] = (torch.rand(e, n, device=DEVICE, generator=gen) + 0.5) * (4.0 / 127.0) * k ** -0.5
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
    dtype = TYPES[case["dtype"]]
    code = int({"f32": rr.ScalarType.kFp32, "f16": rr.ScalarType.kFp16, "bf16": rr.ScalarType.kBf16}[case["dtype"]])
    stream = torch.cuda.current_stream().cuda_stream
    keep = state["buffers"] = {}
    calls = state["calls"] = []
    p = {name: t.data_ptr() for name, t in inp.items() if isinstance(t, torch.Tensor)}

    def new(name, *shape, dtype=dtype):
        keep[name] = torch.empty(*shape, dtype=dtype, device=DEVICE)
        return keep[name].data_ptr()

    def call(entry, args, workspace_size=None):
        size = workspace_size(args) if workspace_size else 0
        workspace = torch.empty(size, dtype=torch.uint8, device=DEVICE) if size else None
        keep["workspace%d" % len(calls)] = workspace
        calls.append((entry, args, rr.RuntimeContext(stream=stream, workspace_bytes=size,
                                                     workspace=workspace.data_ptr() if size else None)))

    k = case["hidden"]
    if case["op"] == "norm":
        t, every = case["tokens"], case["gate_tokens"]
        common = dict(block=p["y"], post_weight=p.get("w_post"), gate=p.get("gate"), gate_tokens=every,
                      pre_weight=p["w_pre"], residual_scale=SCALE, eps=EPS, tokens=t, hidden=k, dtype=code,
                      block_dtype=code)
        h = new("h", t, k)
        call(rr.block_norm, rr.BlockNormArgs(x=p["x"], h=h, n=new("n", t, k), **common))
        outputs = ["h", "n"]
        if case["train"]:
            grads = dict(dx=new("dx", t, k), dblock=new("dy", t, k), dpre_weight=new("dw_pre", k))
            outputs += ["dx", "dy", "dw_pre"]
            if case["post"]:
                grads["dpost_weight"] = new("dw_post", k)
                outputs.append("dw_post")
            if every:
                grads["dgate"] = new("dgate", *inp["gate"].shape)
                outputs.append("dgate")
            call(rr.block_norm_backward, rr.BlockNormBackwardArgs(h=h, dh=p["dh"], dn=p["dn"], **grads, **common),
                 rr.get_block_norm_backward_workspace_size)
    elif case["op"] == "ffn":
        r, f, train = case["rows"], case["inner"], case["train"]
        act = int({"silu": rr.Activation.kSilu, "gelu": rr.Activation.kGeluTanh}[case["act"]])
        common = dict(x=p["x"], w_gate=p["w_gate"], w_up=p["w_up"], w_down=p["w_down"], offsets=p["offsets"],
                      act=new("act", r, f), rows=r, experts=case["experts"], hidden=k, inner=f, output=k,
                      activation=act, dtype=code)
        if train:
            common.update(gate=new("gate", r, f), up=new("up", r, f))
        call(rr.gated_ffn, rr.GatedFfnArgs(y=new("y", r, k), y_dtype=code, **common), rr.get_gated_ffn_workspace_size)
        outputs = ["y"]
        if train:
            grads = {"d" + name: new("d" + name, *inp[name].shape) for name in ("x", "w_gate", "w_up", "w_down")}
            outputs += list(grads)
            call(rr.gated_ffn_backward, rr.GatedFfnBackwardArgs(dy=p["dy"], **grads, **common),
                 rr.get_gated_ffn_backward_workspace_size)
    else:
        r, n = case["rows"], case["output"]
        q, s = new("q", r, k, dtype=torch.int8), new("q_scale", r, dtype=torch.float32)
        call(rr.quantize_rows, rr.QuantizeRowsArgs(x=p["x"], q=q, scale=s, rows=r, hidden=k, dtype=code))
        weights = (dict(w=p["w_gate"], w_scale=p["w_gate_scale"], w_up=p["w_up"], w_up_scale=p["w_up_scale"],
                        activation=int(rr.Activation.kSilu)) if case["gated"]
                   else dict(w=p["w"], w_scale=p["w_scale"]))
        call(rr.int8_grouped_gemm,
             rr.Int8GroupedGemmArgs(q=q, q_scale=s, offsets=p["offsets"], y=new("y", r, n), rows=r,
                                    experts=case["experts"], hidden=k, output=n, dtype=code, **weights),
             rr.get_int8_grouped_gemm_workspace_size)
        outputs = ["y"]
    state["outputs"] = {name: keep[name] for name in outputs}


# ---- the plain forms ----

def _segments(counts):
    row = 0
    for expert, rows in enumerate(counts):
        if rows:
            yield expert, slice(row, row + rows)
        row += rows


def _activation(name: str, g):
    """act(g) and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_ffn(case: dict, inp: dict) -> dict:
    dtype = inp["x"].dtype
    out = {"y": torch.zeros_like(inp["x"])}
    if case["train"]:
        out["dx"] = torch.zeros_like(inp["x"])
        for name in ("w_gate", "w_up", "w_down"):
            out["d" + name] = torch.zeros_like(inp[name])
    for e, rows in _segments(inp["counts"]):
        x = inp["x"][rows].float()
        wg, wu, wd = inp["w_gate"][e].float(), inp["w_up"][e].float(), inp["w_down"][e].float()
        g, u = x @ wg, x @ wu
        s, ds = _activation(case["act"], g)
        a = s * u
        out["y"][rows] = (a @ wd).to(dtype)
        if case["train"]:
            dy = inp["dy"][rows].float()
            da = dy @ wd.t()
            dg, du = da * u * ds, da * s
            out["dx"][rows] = (dg @ wg.t() + du @ wu.t()).to(dtype)
            out["dw_gate"][e] = (x.t() @ dg).to(dtype)
            out["dw_up"][e] = (x.t() @ du).to(dtype)
            out["dw_down"][e] = (a.t() @ dy).to(dtype)
    return out


def _plain_norm(case: dict, inp: dict) -> dict:
    dtype = inp["x"].dtype
    x, y, w_pre = inp["x"].float(), inp["y"].float(), inp["w_pre"].float()
    every, t = case["gate_tokens"], case["tokens"]
    ry = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) if case["post"] else None
    w_post = inp["w_post"].float() if case["post"] else None
    b = y * ry * w_post if case["post"] else y
    group = torch.arange(t, device=DEVICE) // every if every else None
    g = inp["gate"].float()[group] if every else 1.0
    h = x + SCALE * g * b
    rh = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    out = {"h": h.to(dtype), "n": (h * rh * w_pre).to(dtype)}
    if case["train"]:
        dh, dn = inp["dh"].float(), inp["dn"].float()
        v = dn * w_pre
        dh = dh + rh * (v - h * rh * rh * (v * h).mean(1, keepdim=True))
        out["dx"] = dh.to(dtype)
        db = SCALE * g * dh
        if case["post"]:
            v = db * w_post
            out["dy"] = (ry * (v - y * ry * ry * (v * y).mean(1, keepdim=True))).to(dtype)
        else:
            out["dy"] = db.to(dtype)
        out["dw_pre"] = (dn * h * rh).sum(0).to(dtype)
        if case["post"]:
            out["dw_post"] = (db * y * ry).sum(0).to(dtype)
        if every:
            groups, hidden = inp["gate"].shape
            dg = torch.zeros(groups * every, hidden, device=DEVICE)
            dg[:t] = SCALE * dh * b
            out["dgate"] = dg.view(groups, every, hidden).sum(1).to(dtype)
    return out


def _plain_int8(case: dict, inp: dict) -> dict:
    x = inp["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127.0
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))
    y = torch.zeros(case["rows"], case["output"], dtype=inp["x"].dtype, device=DEVICE)
    for e, rows in _segments(inp["counts"]):
        def product(name):
            return (q[rows] @ inp[name][e].float().t()) * scale[rows] * inp[name + "_scale"][e]
        if case["gated"]:
            y[rows] = (_activation("silu", product("w_gate"))[0] * product("w_up")).to(y.dtype)
        else:
            y[rows] = product("w").to(y.dtype)
    return {"y": y}


_PLAIN = {"ffn": _plain_ffn, "norm": _plain_norm, "int8": _plain_int8}


def run(state: dict) -> dict:
    if not state["own"]:
        return _PLAIN[state["case"]["op"]](state["case"], state["inputs"])
    for entry, args, context in state["calls"]:
        status = entry(args, context)
        if not status.ok():
            raise RuntimeError(status.message)
    return state["outputs"]


def work(case: dict) -> dict:
    """Each input read once and each output written once (weights of experts
    with rows), and the products' multiply-adds."""
    size = 4 if case["dtype"] == "f32" else 2
    k = case["hidden"]
    if case["op"] == "norm":
        t, every = case["tokens"], case["gate_tokens"]
        gates = (t + every - 1) // every * k if every else 0
        values = 4 * t * k + gates + 2 * k
        flops = 12 * t * k
        if case["train"]:
            values += 4 * t * k + gates + 2 * k  # dh, dn, dx, dy, and the gradients of gate and weights
            flops += 30 * t * k
        return {"bytes": size * values, "flops": flops}
    r, active = case["rows"], case["active"]
    if case["op"] == "ffn":
        f = case["inner"]
        values, flops = 2 * r * k + 3 * active * k * f, 6 * r * k * f
        if case["train"]:
            values += 2 * r * k + 3 * case["experts"] * k * f
            flops *= 3
        return {"bytes": size * values + 4 * (case["experts"] + 1), "flops": flops}
    n, weights = case["output"], 2 if case["gated"] else 1
    return {"bytes": size * (r * k + r * n) + active * weights * n * (k + 4) + 4 * (case["experts"] + 1),
            "flops": 2 * weights * r * k * n}


# ---- results in 64 bits ----

def exact(case: dict, seed: int):
    inp = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, inp)
    if case["op"] == "ffn":
        return _exact_ffn(case, inp)
    # the quantised rows are whole numbers of the 32-bit quotients; everything after them is exact in 64 bits
    x = inp["x"].cpu().numpy() if inp["x"].dtype != torch.bfloat16 else inp["x"].float().cpu().numpy()
    x = x.astype(np.float32)
    scale = np.abs(x).max(axis=1, keepdims=True) / np.float32(127.0)
    q = np.rint(np.divide(x, scale, out=np.zeros_like(x), where=scale > 0))
    q = torch.from_numpy(q).to(DEVICE).double()
    scale = torch.from_numpy(scale).to(DEVICE).double()
    y = torch.zeros(case["rows"], case["output"], dtype=torch.float64, device=DEVICE)
    first = 0
    for e, count in enumerate(inp["counts"]):
        last = first + count
        parts = [(q[first:last] @ inp[w][e].double().t().contiguous()) * scale[first:last] * inp[w + "_scale"][e].double()
                 for w in (("w_gate", "w_up") if case["gated"] else ("w",))]
        y[first:last] = parts[0] * torch.sigmoid(parts[0]) * parts[1] if case["gated"] else parts[0]
        first = last
    return {"y": y}


def _exact_ffn(case: dict, inp: dict) -> dict:
    """By differentiating the block's formula in float64."""
    def act(g):
        if case["act"] == "silu":
            return g * torch.sigmoid(g)
        return g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))  # (1 + tanh z) / 2

    names = ("w_gate", "w_up", "w_down")
    f64 = dict(dtype=torch.float64, device=DEVICE)
    out = {"y": torch.zeros(inp["x"].shape, **f64)}
    if case["train"]:
        out["dx"] = torch.zeros(inp["x"].shape, **f64)
        for name in names:
            out["d" + name] = torch.zeros(inp[name].shape, **f64)
    first = 0
    for e, count in enumerate(inp["counts"]):
        if not count:
            continue
        rows = slice(first, first + count)
        first += count
        x, wg, wu, wd = (t.double().requires_grad_(case["train"])
                         for t in (inp["x"][rows], *(inp[name][e] for name in names)))
        y = (act(x @ wg) * (x @ wu)) @ wd
        out["y"][rows] = y.detach()
        if case["train"]:
            grads = torch.autograd.grad(y, (x, wg, wu, wd), inp["dy"][rows].double())
            out["dx"][rows] = grads[0]
            for name, grad in zip(names, grads[1:]):
                out["d" + name][e] = grad
    return out


def _exact_norm(case: dict, inp: dict) -> dict:
    """By differentiating the operator's formula in float64."""
    v = {name: t.double().requires_grad_(case["train"]) for name, t in inp.items()}

    def norm(a, w):
        return a / torch.sqrt(a.square().mean(dim=1, keepdim=True) + EPS) * w

    b = norm(v["y"], v["w_post"]) if case["post"] else v["y"]
    if case["gate_tokens"]:
        b = b * v["gate"].repeat_interleave(case["gate_tokens"], dim=0)[:case["tokens"]]
    h = v["x"] + SCALE * b
    n = norm(h, v["w_pre"])
    out = {"h": h.detach(), "n": n.detach()}
    if case["train"]:
        names = ["x", "y", "w_pre"] + ["w_post"] * case["post"] + ["gate"] * (case["gate_tokens"] > 0)
        grads = torch.autograd.grad((h, n), [v[name] for name in names], (inp["dh"].double(), inp["dn"].double()))
        for name, grad in zip(names, grads):
            out["dgate" if name == "gate" else "d" + name] = grad
    return out
