"""A mixture-of-experts block on the library's operators: forward, backward and int8 serving.

    n      = N(x; pre)                                    block_norm
    routes = top-2 of softmax(n router)                   dense_gemm, topk_gate,
             rows of n in order of their experts          histogram_exclusive_scan, token_permute
    r      = act(rows Wg) * (rows Wu) Wd                  gated_ffn (or quantize_rows, int8_grouped_gemm)
    y      = sum over a token's routes of weight * r      unpermute
    h      = x + scale * N(y; post),  n' = N(h; next)     block_norm

The routing chain computes in FP32, the experts in BF16 (or int8): rows are cast where
they enter the experts, whose results are FP32 again. The backward pass takes the routing
weights as constants. Run `python examples/moe_block.py` for its times on a GPU.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import raggedroute_amd as rr  # noqa: E402

FP32, BF16 = int(rr.ScalarType.kFp32), int(rr.ScalarType.kBf16)
TOP_K = 2


def call(operator, args, workspace_size=None):
    """Runs an operator on torch's current stream, with the workspace it asks for."""
    size = workspace_size(args) if workspace_size is not None else 0
    workspace = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    context = rr.RuntimeContext(stream=torch.cuda.current_stream().cuda_stream, workspace=workspace.data_ptr(),
                                workspace_bytes=size, architecture=int(rr.DeviceArchitecture.kGfx950))
    status = operator(args, context)
    if not status.ok():
        raise RuntimeError(repr(status))


def empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


class MoeBlock:
    """Weights of one block: norms and router in FP32, experts in BF16 and, after
    `quantize`, in int8."""

    def __init__(self, hidden, inner, experts, seed=0, scale=0.5, eps=1e-6):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def normal(*shape, dtype=torch.float32):
            t = torch.randn(shape, device="cuda", generator=gen)
            return (t * shape[-2] ** -0.5).to(dtype)

        self.hidden, self.inner, self.experts, self.scale, self.eps = hidden, inner, experts, scale, eps
        self.router = normal(hidden, experts)
        self.w_gate = normal(experts, hidden, inner, dtype=torch.bfloat16)
        self.w_up = normal(experts, hidden, inner, dtype=torch.bfloat16)
        self.w_down = normal(experts, inner, hidden, dtype=torch.bfloat16)
        self.pre, self.post, self.next = (1 + 0.1 * torch.randn(hidden, device="cuda", generator=gen) for _ in range(3))

    # ---- the parts ----
    def norm(self, x, weight, block=None, post=None):
        """h = x + scale * N(block; post) (x without a block) and N(h; weight)."""
        tokens = x.shape[0]
        n, h = torch.empty_like(x), torch.empty_like(x) if block is not None else None
        call(rr.block_norm, rr.BlockNormArgs(
            x=x.data_ptr(), block=block.data_ptr() if block is not None else None,
            post_weight=post.data_ptr() if post is not None else None, pre_weight=weight.data_ptr(),
            h=h.data_ptr() if h is not None else None, n=n.data_ptr(), residual_scale=self.scale, eps=self.eps,
            gate_tokens=1, tokens=tokens, hidden=self.hidden, dtype=FP32, block_dtype=FP32),
            rr.get_block_norm_workspace_size)
        return h, n

    def route(self, n):
        """Top-2 experts of every token and its rows in their order."""
        tokens, routes = n.shape[0], TOP_K * n.shape[0]
        int32 = dict(dtype=torch.int32)
        logits, ids, weights = empty(tokens, self.experts), empty(tokens, TOP_K, **int32), empty(tokens, TOP_K)
        counts, offsets = empty(self.experts, **int32), empty(self.experts + 1, **int32)
        rows, position, route = empty(routes, self.hidden), empty(routes, **int32), empty(routes, **int32)
        call(rr.dense_gemm, rr.DenseGemmArgs(
            a=rr.cview(n.data_ptr()), b=rr.cview(self.router.data_ptr()), c=rr.mview(logits.data_ptr()), m=tokens,
            n=self.experts, k=self.hidden), rr.get_dense_gemm_workspace_size)
        call(rr.topk_gate, rr.TopKGateArgs(
            logits=rr.cview(logits.data_ptr()), expert_ids=ids.data_ptr(), weights=rr.mview(weights.data_ptr()),
            tokens=tokens, experts=self.experts), rr.get_topk_gate_workspace_size)
        call(rr.histogram_exclusive_scan, rr.HistogramExclusiveScanArgs(
            expert_ids=ids.data_ptr(), counts=counts.data_ptr(), offsets=offsets.data_ptr(), route_pairs=routes,
            experts=self.experts), rr.get_histogram_exclusive_scan_workspace_size)
        call(rr.token_permute, rr.TokenPermuteArgs(
            x=rr.cview(n.data_ptr()), expert_ids=ids.data_ptr(), offsets=offsets.data_ptr(),
            x_permuted=rr.mview(rows.data_ptr()), route_pos=position.data_ptr(), sorted_route=route.data_ptr(),
            tokens=tokens, experts=self.experts, top_k=TOP_K, hidden=self.hidden), rr.get_token_permute_workspace_size)
        return dict(rows=rows, ids=ids, weights=weights, offsets=offsets, position=position, route=route)

    def unroute(self, r, routes):
        tokens = routes["ids"].shape[0]
        y = empty(tokens, self.hidden)
        call(rr.unpermute, rr.UnpermuteArgs(
            y_permuted=rr.cview(r.data_ptr()), route_pos=routes["position"].data_ptr(),
            route_weights=rr.cview(routes["weights"].data_ptr()), y=rr.mview(y.data_ptr()), tokens=tokens,
            top_k=TOP_K, output=self.hidden), rr.get_unpermute_workspace_size)
        return y

    # ---- the block ----
    def forward(self, x, keep=False):
        """h and the next block's input; with `keep` also what `backward` reads."""
        _, n = self.norm(x, self.pre)
        routes = self.route(n)
        rows = routes["rows"].to(torch.bfloat16)
        count = rows.shape[0]
        gate, up = (empty(count, self.inner, dtype=torch.bfloat16) if keep else None for _ in range(2))
        act, r = empty(count, self.inner, dtype=torch.bfloat16), empty(count, self.hidden)
        call(rr.gated_ffn, rr.GatedFfnArgs(
            x=rows.data_ptr(), w_gate=self.w_gate.data_ptr(), w_up=self.w_up.data_ptr(),
            w_down=self.w_down.data_ptr(), offsets=routes["offsets"].data_ptr(),
            gate=gate.data_ptr() if keep else None, up=up.data_ptr() if keep else None, act=act.data_ptr(),
            y=r.data_ptr(), rows=count, experts=self.experts, hidden=self.hidden, inner=self.inner,
            output=self.hidden, activation=int(rr.Activation.kSilu), dtype=BF16, y_dtype=FP32),
            rr.get_gated_ffn_workspace_size)
        y = self.unroute(r, routes)
        h, n_next = self.norm(x, self.next, y, self.post)
        kept = dict(x=x, rows=rows, gate=gate, up=up, act=act, y=y, h=h, routes=routes) if keep else None
        return h, n_next, kept

    def norm_backward(self, h, weight, dh, dn, block=None, post=None):
        grad = {"dx": torch.empty_like(h)}
        grad["dpre"] = torch.empty_like(weight) if dn is not None else None
        grad["dblock"] = torch.empty_like(block) if block is not None else None
        grad["dpost"] = torch.empty_like(post) if post is not None else None

        def at(t):
            return t.data_ptr() if t is not None else None

        call(rr.block_norm_backward, rr.BlockNormBackwardArgs(
            h=h.data_ptr(), block=at(block), post_weight=at(post), pre_weight=weight.data_ptr(), dh=at(dh), dn=at(dn),
            dx=at(grad["dx"]), dblock=at(grad["dblock"]), dpre_weight=at(grad["dpre"]), dpost_weight=at(grad["dpost"]),
            residual_scale=self.scale, eps=self.eps, gate_tokens=1, tokens=h.shape[0], hidden=self.hidden, dtype=FP32,
            block_dtype=FP32), rr.get_block_norm_backward_workspace_size)
        return grad

    def backward(self, kept, dh, dn_next):
        """Gradients of x and of every weight but the router's."""
        last = self.norm_backward(kept["h"], self.next, dh, dn_next, kept["y"], self.post)
        routes, rows = kept["routes"], kept["rows"]
        route = routes["route"].long()
        # a route's result enters its token's sum with the routing weight
        dr = (last["dblock"][route // TOP_K] * routes["weights"].flatten()[route][:, None]).to(torch.bfloat16)
        dx, dw_gate, dw_up, dw_down = (torch.empty_like(t) for t in (rows, self.w_gate, self.w_up, self.w_down))
        call(rr.gated_ffn_backward, rr.GatedFfnBackwardArgs(
            x=rows.data_ptr(), w_gate=self.w_gate.data_ptr(), w_up=self.w_up.data_ptr(),
            w_down=self.w_down.data_ptr(), offsets=routes["offsets"].data_ptr(), gate=kept["gate"].data_ptr(),
            up=kept["up"].data_ptr(), act=kept["act"].data_ptr(), dy=dr.data_ptr(), dx=dx.data_ptr(),
            dw_gate=dw_gate.data_ptr(), dw_up=dw_up.data_ptr(), dw_down=dw_down.data_ptr(), rows=rows.shape[0],
            experts=self.experts, hidden=self.hidden, inner=self.inner, output=self.hidden,
            activation=int(rr.Activation.kSilu), dtype=BF16), rr.get_gated_ffn_backward_workspace_size)
        # a token's norm fed its top-2 routes' rows
        dn = dx.float()[routes["position"].long()].view(-1, TOP_K, self.hidden).sum(1)
        first = self.norm_backward(kept["x"], self.pre, last["dx"], dn)
        return dict(x=first["dx"], pre=first["dpre"], post=last["dpost"], next=last["dpre"], w_gate=dw_gate, w_up=dw_up,
                    w_down=dw_down)

    # ---- serving in int8 ----
    @staticmethod
    def to_int8(x):
        """Rows of x (any leading shape) with a scale each."""
        q, scale = torch.empty(x.shape, dtype=torch.int8, device="cuda"), empty(*x.shape[:-1])
        call(rr.quantize_rows, rr.QuantizeRowsArgs(
            x=x.data_ptr(), q=q.data_ptr(), scale=scale.data_ptr(), rows=scale.numel(), hidden=x.shape[-1],
            dtype=FP32 if x.dtype == torch.float32 else BF16), rr.get_quantize_rows_workspace_size)
        return q, scale

    def quantize(self):
        """Lays the experts out in int8: a row per expert and output channel."""
        self.q_gate, self.q_up, self.q_down = (self.to_int8(w.transpose(1, 2).contiguous())
                                               for w in (self.w_gate, self.w_up, self.w_down))

    def int8_product(self, rows, weight, routes, dtype, up=None):
        q, scale = self.to_int8(rows)
        output = weight[0].shape[1]
        y = empty(rows.shape[0], output, dtype=dtype)
        call(rr.int8_grouped_gemm, rr.Int8GroupedGemmArgs(
            q=q.data_ptr(), q_scale=scale.data_ptr(), w=weight[0].data_ptr(), w_scale=weight[1].data_ptr(),
            w_up=up[0].data_ptr() if up else None, w_up_scale=up[1].data_ptr() if up else None,
            offsets=routes["offsets"].data_ptr(), y=y.data_ptr(), rows=rows.shape[0], experts=self.experts,
            hidden=rows.shape[1], output=output, activation=int(rr.Activation.kSilu),
            dtype=FP32 if dtype == torch.float32 else BF16), rr.get_int8_grouped_gemm_workspace_size)
        return y

    def forward_int8(self, x):
        _, n = self.norm(x, self.pre)
        routes = self.route(n)
        act = self.int8_product(routes["rows"], self.q_gate, routes, torch.bfloat16, self.q_up)
        r = self.int8_product(act, self.q_down, routes, torch.float32)
        return self.norm(x, self.next, self.unroute(r, routes), self.post)


def main():
    block = MoeBlock(hidden=1024, inner=512, experts=64)
    block.quantize()
    for tokens in (1, 64, 4096):
        x = torch.randn(tokens, block.hidden, device="cuda")
        dh, dn = torch.randn_like(x), torch.randn_like(x)

        def step():
            block.backward(block.forward(x, keep=True)[2], dh, dn)

        exact, quick = block.forward(x)[0], block.forward_int8(x)[0]
        away = ((quick - exact).norm() / (exact - x).norm()).item()
        print(f"{tokens} tokens: int8 moves the block's addition by {away:.3f} of its norm")
        for name, run in (("forward", lambda: block.forward(x)), ("forward, int8", lambda: block.forward_int8(x)),
                          ("forward and backward", step)):
            for _ in range(3):
                run()
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(10):
                run()
            end.record()
            torch.cuda.synchronize()
            print(f"  {name:24s}{begin.elapsed_time(end) * 100:9.1f} us")


if __name__ == "__main__":
    main()
