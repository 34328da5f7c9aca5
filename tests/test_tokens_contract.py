"""Refusals and workspace queries of the entries that take tokens to their experts and back,
and of the 4-bit ones (no device call is made)."""
from __future__ import annotations

import ctypes

import pytest

import raggedroute_amd as rr

S = rr.StatusCode
GFX950 = int(rr.DeviceArchitecture.kGfx950)
P = 4096  # a pointer that is never followed


def ctx(**kw):
    return rr.RuntimeContext(**({"architecture": GFX950} | kw))


ENTRIES = {
    "sort_tokens": (rr.SortTokensArgs, dict(x=P, expert_ids=P, offsets=P, route_pos=P, sorted_route=P, x_sorted=P,
                                            tokens=4, experts=3, top_k=2, hidden=8)),
    "sort_tokens_backward": (rr.SortTokensBackwardArgs, dict(dx_sorted=P, route_pos=P, dx=P, tokens=4, top_k=2, hidden=8)),
    "combine_tokens": (rr.CombineTokensArgs, dict(y_sorted=P, route_pos=P, route_weights=P, y=P, tokens=4, top_k=2,
                                                  hidden=8)),
    "combine_tokens_backward": (rr.CombineTokensBackwardArgs,
                                dict(dy=P, y_sorted=P, route_pos=P, route_weights=P, dy_sorted=P, droute_weights=P,
                                     tokens=4, top_k=2, hidden=8)),
    "topk_gate_backward": (rr.TopKGateBackwardArgs, dict(expert_ids=P, weights=P, dweights=P, dlogits=P, tokens=4,
                                                         experts=3, top_k=2)),
    "quantize_rows_mxfp4": (rr.QuantizeRowsMxfp4Args, dict(x=P, sorted_route=P, q=P, scale=P, rows=8, hidden=8, tokens=4,
                                                           top_k=2)),
    "mxfp4_grouped_gemm": (rr.Mxfp4GroupedGemmArgs, dict(q=P, q_scale=P, w=P, w_scale=P, w_up=P, w_up_scale=P, offsets=P,
                                                         y=P, rows=4, experts=2, hidden=8, output=8)),
}


def refusal(name, context=None, **change):
    args, good = ENTRIES[name]
    status = getattr(rr, name)(args(**(good | change)), context or ctx())
    assert not status.ok() and status.message
    return status.code


@pytest.mark.parametrize("name", list(ENTRIES))
def test_missing_structs(name):
    fn = getattr(rr.lib, "rr_" + name)
    assert fn(None, ctx()).code == S.kInvalidArgument
    assert fn(ENTRIES[name][0](**ENTRIES[name][1]), None).code == S.kInvalidArgument


WIDTH = [0, -1, (1 << 20) + 1]
ROUTES = dict(tokens=[-1, 1 << 30], top_k=[0, -1, 65])
SIZES = {
    "sort_tokens": dict(experts=[0, 1025], hidden=WIDTH, **ROUTES),
    "sort_tokens_backward": dict(hidden=WIDTH, **ROUTES),
    "combine_tokens": dict(hidden=WIDTH, **ROUTES),
    "combine_tokens_backward": dict(hidden=WIDTH, **ROUTES),
    "topk_gate_backward": dict(experts=[0, 1025], **ROUTES),
    "quantize_rows_mxfp4": dict(rows=[-1], hidden=WIDTH, **ROUTES),
    "mxfp4_grouped_gemm": dict(rows=[-1], experts=[0, 1025], hidden=WIDTH, output=WIDTH, activation=[2, -1]),
}


@pytest.mark.parametrize("name", list(ENTRIES))
def test_sizes(name):
    for field, values in SIZES[name].items():
        for value in values:
            assert refusal(name, **{field: value}) == S.kInvalidArgument, (field, value)


@pytest.mark.parametrize("name", list(ENTRIES))
def test_types_architecture_family(name):
    if name != "topk_gate_backward":
        assert refusal(name, dtype=int(rr.ScalarType.kFp8E4M3)) == S.kUnsupportedDataType
    other = {"sort_tokens": "x_dtype", "sort_tokens_backward": "x_dtype", "combine_tokens": "y_dtype",
             "combine_tokens_backward": "y_dtype"}.get(name)
    if other:
        assert refusal(name, **{other: int(rr.ScalarType.kFp16)}) == S.kUnsupportedDataType
        assert refusal(name, dtype=int(rr.ScalarType.kFp32), **{other: int(rr.ScalarType.kBf16)}) == S.kUnsupportedDataType
    for arch in (rr.DeviceArchitecture.kOther, rr.DeviceArchitecture.kSm86):
        assert refusal(name, ctx(architecture=int(arch))) == S.kUnsupportedArchitecture
    F = rr.KernelFamily
    for kernel in (rr.kernel(F.kAuto, 1), rr.kernel(F.kOptimized, 0), rr.kernel(F.kOptimized, 1), rr.kernel(F.kNaive, 1),
                   rr.KernelSelection(7, 0)):
        assert refusal(name, kernel=kernel) == S.kUnsupportedKernelVariant
    if name != "mxfp4_grouped_gemm":
        assert refusal(name, kernel=rr.kernel(F.kNaive)) == S.kUnsupportedKernelVariant


OPTIONAL = {
    "sort_tokens": ["sorted_route", "x_sorted"],
    "sort_tokens_backward": [],
    "combine_tokens": ["route_weights"],
    "combine_tokens_backward": ["route_weights", "dy_sorted", "droute_weights"],
    "topk_gate_backward": [],
    "quantize_rows_mxfp4": ["sorted_route"],
    "mxfp4_grouped_gemm": ["w_up"],
}


@pytest.mark.parametrize("name", list(ENTRIES))
def test_pointers(name):
    for field, value in ENTRIES[name][1].items():
        if value != P:
            continue
        if field not in OPTIONAL[name]:
            assert refusal(name, **{field: None}) == S.kInvalidArgument, field
        assert refusal(name, **{field: P + 1}) == S.kInvalidArgument, field


def test_alignment_of_packed_rows():
    for field in ("q", "w", "w_up"):
        assert refusal("mxfp4_grouped_gemm", **{field: P + 8}) == S.kInvalidArgument
    for field in ("q_scale", "w_scale", "w_up_scale"):
        assert refusal("mxfp4_grouped_gemm", **{field: P + 4}) == S.kInvalidArgument
    assert refusal("quantize_rows_mxfp4", q=P + 8) == S.kInvalidArgument
    assert refusal("quantize_rows_mxfp4", scale=P + 4) == S.kInvalidArgument


def test_workspaces():
    for name, (args, good) in ENTRIES.items():
        assert getattr(rr, f"get_{name}_workspace_size")(args(**good)) == 0, name
        assert getattr(rr.lib, f"rr_{name}_workspace_size")(None) == 0, name


def test_workspace_of_many_routes():
    """The counts of 32 parts of the routes."""
    def args(**change):
        return rr.SortTokensArgs(**(ENTRIES["sort_tokens"][1] | change))

    for tokens, top_k, experts, need in ((4096, 2, 256, 0), (8193, 1, 256, 32 * 256 * 4), (2 ** 30, 1, 9, 32 * 9 * 4),
                                         (2 ** 30, 1, 1024, 32 * 1024 * 4), (2 ** 30, 2, 9, 0), (-1, 2, 9, 0)):
        assert rr.get_sort_tokens_workspace_size(args(tokens=tokens, top_k=top_k, experts=experts)) == need
    many = dict(tokens=8193, top_k=1, experts=9)
    size = 32 * 9 * 4
    assert refusal("sort_tokens", **many) == S.kInsufficientWorkspace
    assert refusal("sort_tokens", ctx(workspace=P, workspace_bytes=size - 1), **many) == S.kInsufficientWorkspace
    assert refusal("sort_tokens", ctx(workspace=P + 4, workspace_bytes=size), **many) == S.kInvalidArgument


def test_nothing_to_do():
    for name, change in (("sort_tokens_backward", dict(tokens=0)), ("combine_tokens", dict(tokens=0)),
                         ("combine_tokens_backward", dict(tokens=0)),
                         ("combine_tokens_backward", dict(dy_sorted=None, droute_weights=None)),
                         ("topk_gate_backward", dict(tokens=0)), ("quantize_rows_mxfp4", dict(rows=0)),
                         ("quantize_rows_mxfp4", dict(tokens=0)), ("mxfp4_grouped_gemm", dict(rows=0))):
        args, good = ENTRIES[name]
        assert getattr(rr, name)(args(**(good | change)), ctx()).ok(), name


def test_struct_sizes():
    # C struct sizes on LP64, from the header's field lists
    for name, size in (("sort_tokens", 6 * 8 + 6 * 4 + 8), ("sort_tokens_backward", 3 * 8 + 5 * 4 + 8 + 4),
                       ("combine_tokens", 4 * 8 + 5 * 4 + 8 + 4), ("combine_tokens_backward", 6 * 8 + 5 * 4 + 8 + 4),
                       ("topk_gate_backward", 4 * 8 + 3 * 4 + 8 + 4), ("quantize_rows_mxfp4", 4 * 8 + 5 * 4 + 8 + 4),
                       ("mxfp4_grouped_gemm", 8 * 8 + 6 * 4 + 8)):
        assert ctypes.sizeof(ENTRIES[name][0]) == size, name
