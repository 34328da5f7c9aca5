"""Refusals and workspace queries of the expert block's entries (no device call is made)."""
from __future__ import annotations

import pytest

import raggedroute_amd as rr

S = rr.StatusCode
GFX950 = int(rr.DeviceArchitecture.kGfx950)
P = 4096  # a pointer that is never followed


def ctx(**kw):
    return rr.RuntimeContext(**({"architecture": GFX950} | kw))


FFN = dict(x=P, w_gate=P, w_up=P, w_down=P, offsets=P, act=P, y=P, rows=4, experts=2, hidden=8, inner=8, output=8)
BACK = dict(x=P, w_gate=P, w_up=P, w_down=P, offsets=P, gate=P, up=P, act=P, dy=P, dx=P, dw_gate=P, dw_up=P, dw_down=P,
            rows=4, experts=2, hidden=8, inner=8, output=8)
NORM = dict(x=P, block=P, post_weight=P, gate=P, gate_tokens=1, pre_weight=P, h=P, n=P, tokens=4, hidden=8)
NORM_BACK = dict(h=P, block=P, post_weight=P, gate=P, gate_tokens=1, pre_weight=P, dh=P, dn=P, dx=P, dblock=P, dgate=P,
                 dpre_weight=P, dpost_weight=P, tokens=4, hidden=8)
QUANT = dict(x=P, q=P, scale=P, rows=4, hidden=8)
INT8 = dict(q=P, q_scale=P, w=P, w_scale=P, offsets=P, y=P, rows=4, experts=2, hidden=8, output=8)

ENTRIES = {
    "gated_ffn": (rr.gated_ffn, rr.GatedFfnArgs, FFN),
    "gated_ffn_backward": (rr.gated_ffn_backward, rr.GatedFfnBackwardArgs, BACK),
    "block_norm": (rr.block_norm, rr.BlockNormArgs, NORM),
    "block_norm_backward": (rr.block_norm_backward, rr.BlockNormBackwardArgs, NORM_BACK),
    "quantize_rows": (rr.quantize_rows, rr.QuantizeRowsArgs, QUANT),
    "int8_grouped_gemm": (rr.int8_grouped_gemm, rr.Int8GroupedGemmArgs, INT8),
}


def refusal(name, context=None, **change):
    entry, args, good = ENTRIES[name]
    status = entry(args(**(good | change)), context or ctx())
    assert not status.ok() and status.message
    return status.code


@pytest.mark.parametrize("name", list(ENTRIES))
def test_missing_structs(name):
    fn = getattr(rr.lib, "rr_" + name)
    assert fn(None, ctx()).code == S.kInvalidArgument
    assert fn(ENTRIES[name][1](**ENTRIES[name][2]), None).code == S.kInvalidArgument


SIZES = {
    "gated_ffn": dict(rows=[-1], experts=[0, -1, 1025], hidden=[0, -1, 1 << 21], inner=[0, 1 << 21], output=[0, 1 << 21]),
    "gated_ffn_backward": dict(rows=[-1], experts=[0, 1025], hidden=[0, 1 << 21], inner=[0, 1 << 21], output=[0, 1 << 21]),
    "block_norm": dict(tokens=[-1], hidden=[0, -1, 1 << 21], gate_tokens=[0, -1], eps=[0.0, -1.0, float("nan")]),
    "block_norm_backward": dict(tokens=[-1], hidden=[0, 1 << 21], gate_tokens=[0], eps=[0.0, float("nan")]),
    "quantize_rows": dict(rows=[-1], hidden=[0, 1 << 21]),
    "int8_grouped_gemm": dict(rows=[-1], experts=[0, 1025], hidden=[0, 131073], output=[0, 1 << 21]),
}


@pytest.mark.parametrize("name", list(ENTRIES))
def test_sizes(name):
    for field, values in SIZES[name].items():
        for value in values:
            assert refusal(name, **{field: value}) == S.kInvalidArgument, (field, value)


@pytest.mark.parametrize("name", list(ENTRIES))
def test_types_architecture_family(name):
    bad = int(rr.ScalarType.kFp8E4M3)
    assert refusal(name, dtype=bad) == S.kUnsupportedDataType
    if name.startswith("gated"):
        assert refusal(name, dtype=int(rr.ScalarType.kFp32)) == S.kUnsupportedDataType
    if name == "gated_ffn":
        assert refusal(name, y_dtype=int(rr.ScalarType.kFp16)) == S.kUnsupportedDataType
    if name.startswith("block_norm"):
        assert refusal(name, block_dtype=int(rr.ScalarType.kFp16)) == S.kUnsupportedDataType
    for arch in (rr.DeviceArchitecture.kOther, rr.DeviceArchitecture.kSm86):
        assert refusal(name, ctx(architecture=int(arch))) == S.kUnsupportedArchitecture
    F = rr.KernelFamily
    for kernel in (rr.kernel(F.kAuto, 1), rr.kernel(F.kOptimized, 0), rr.kernel(F.kOptimized, 1), rr.kernel(F.kNaive, 1),
                   rr.KernelSelection(7, 0)):
        assert refusal(name, kernel=kernel) == S.kUnsupportedKernelVariant
    if name in ("block_norm", "block_norm_backward", "quantize_rows"):
        assert refusal(name, kernel=rr.kernel(F.kNaive)) == S.kUnsupportedKernelVariant


REQUIRED = {
    "gated_ffn": ["x", "w_gate", "w_up", "w_down", "offsets", "act", "y"],
    "gated_ffn_backward": ["x", "w_gate", "w_up", "w_down", "offsets", "gate", "up", "act", "dy"],
    "block_norm": ["x", "pre_weight", "h"],
    "block_norm_backward": ["h", "pre_weight", "dx"],
    "quantize_rows": ["x", "q", "scale"],
    "int8_grouped_gemm": ["q", "q_scale", "w", "w_scale", "offsets", "y"],
}


@pytest.mark.parametrize("name", list(ENTRIES))
def test_pointers(name):
    for field in REQUIRED[name]:
        assert refusal(name, **{field: None}) == S.kInvalidArgument, field
    for field, value in ENTRIES[name][2].items():
        if value == P and not (name == "int8_grouped_gemm" and field in ("q", "w")) and not (name == "quantize_rows" and field == "q"):
            assert refusal(name, **{field: P + 1}) == S.kInvalidArgument, field


def test_pairs_and_optional_parts():
    assert refusal("gated_ffn", gate=P) == S.kInvalidArgument
    assert refusal("gated_ffn", up=P) == S.kInvalidArgument
    assert refusal("gated_ffn", activation=2) == S.kInvalidArgument
    assert refusal("gated_ffn_backward", dw_up=None) == S.kInvalidArgument
    assert refusal("gated_ffn_backward", activation=-1) == S.kInvalidArgument
    assert refusal("block_norm", n=None, h=None, block=None) == S.kInvalidArgument
    assert refusal("block_norm_backward", dh=None, dn=None) == S.kInvalidArgument
    assert refusal("int8_grouped_gemm", w_up=P) == S.kInvalidArgument
    assert refusal("int8_grouped_gemm", w_up=P, w_up_scale=P, activation=5) == S.kInvalidArgument


def test_workspaces():
    args = rr.GatedFfnBackwardArgs(**BACK)
    need = rr.get_gated_ffn_backward_workspace_size(args)
    assert need == 2 * 4 * 8 * 2
    assert rr.get_gated_ffn_backward_workspace_size(rr.GatedFfnBackwardArgs(**(BACK | dict(rows=1, inner=3)))) == 32
    for name, size in (("gated_ffn_backward", need),
                       ("block_norm_backward", rr.get_block_norm_backward_workspace_size(rr.BlockNormBackwardArgs(**NORM_BACK)))):
        assert size > 0
        assert refusal(name) == S.kInsufficientWorkspace
        assert refusal(name, ctx(workspace=P, workspace_bytes=size - 1)) == S.kInsufficientWorkspace
        assert refusal(name, ctx(workspace=P + 4, workspace_bytes=size)) == S.kInvalidArgument
    assert rr.get_gated_ffn_workspace_size(rr.GatedFfnArgs(**FFN)) == 0
    assert rr.get_gated_ffn_backward_workspace_size(rr.GatedFfnBackwardArgs(**(BACK | dict(rows=0)))) == 0
    assert rr.get_block_norm_backward_workspace_size(rr.BlockNormBackwardArgs(**(NORM_BACK | dict(tokens=0)))) == 0
    # past 32 bits
    assert rr.get_gated_ffn_backward_workspace_size(
        rr.GatedFfnBackwardArgs(**(BACK | dict(rows=1 << 30, inner=1 << 12)))) == 1 << 44


def test_nothing_to_do():
    assert rr.gated_ffn(rr.GatedFfnArgs(rows=0, experts=2, hidden=8, inner=8, output=8), ctx()).ok()
    assert rr.block_norm(rr.BlockNormArgs(tokens=0, hidden=8), ctx()).ok()
    assert rr.quantize_rows(rr.QuantizeRowsArgs(rows=0, hidden=8), ctx()).ok()
    assert rr.int8_grouped_gemm(rr.Int8GroupedGemmArgs(rows=0, experts=2, hidden=8, output=8), ctx()).ok()


def test_struct_sizes():
    import ctypes

    # C struct sizes on LP64, from the header's field lists
    for name, size in (("GatedFfnArgs", 9 * 8 + 8 * 4 + 8), ("GatedFfnBackwardArgs", 13 * 8 + 7 * 4 + 8 + 4),
                       ("BlockNormArgs", 7 * 8 + 7 * 4 + 8 + 4), ("BlockNormBackwardArgs", 12 * 8 + 7 * 4 + 8 + 4),
                       ("QuantizeRowsArgs", 3 * 8 + 3 * 4 + 8 + 4), ("Int8GroupedGemmArgs", 8 * 8 + 6 * 4 + 8)):
        assert ctypes.sizeof(getattr(rr, name)) == size, name
