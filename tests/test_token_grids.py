"""Grids of the operators that take tokens to their experts and back and of the 4-bit products at
the ends of their ranges, by launches that a stand-in for HIP counts (no GPU is used:
tests/cpp/launches.cpp)."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))

PROGRAM = """
import ctypes, sys
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import raggedroute_amd as rr
P = 4096
MOST = 2 ** 31 - 1


def grid(name, args):
    size = getattr(rr, f"get_{name}_workspace_size")(args)
    context = rr.RuntimeContext(architecture=int(rr.DeviceArchitecture.kGfx950), workspace=P, workspace_bytes=size)
    status = getattr(rr, name)(args, context)
    assert status.ok(), status.message
    return hip.launches_grid()


maps = dict(expert_ids=P, offsets=P, route_pos=P, hidden=1)
for tokens, top_k, experts in ((MOST, 1, 256), (MOST // 64, 64, 8), (MOST, 1, 1024), (129, 1, 8), (1, 64, 8)):
    print("maps", tokens, top_k, experts, grid("sort_tokens", rr.SortTokensArgs(tokens=tokens, top_k=top_k, experts=experts, **maps)))
rows = dict(route_pos=P, hidden=1 << 20, dtype=0)
print("combine", grid("combine_tokens", rr.CombineTokensArgs(y_sorted=P, y=P, tokens=MOST, top_k=1, **rows)))
print("backward", grid("combine_tokens_backward", rr.CombineTokensBackwardArgs(
    dy=P, y_sorted=P, dy_sorted=P, droute_weights=P, tokens=MOST, top_k=1, **rows)))
print("gate", grid("topk_gate_backward", rr.TopKGateBackwardArgs(expert_ids=P, weights=P, dweights=P, dlogits=P,
                                                                 tokens=MOST, top_k=1, experts=1024)))
print("quantize", grid("quantize_rows_mxfp4", rr.QuantizeRowsMxfp4Args(x=P, q=P, scale=P, rows=MOST, hidden=1 << 20)))
for rows, experts, output in ((12 * 1024, 1024, 1 << 20), (MOST, 1, 1), (16, 8, 14336), (16384, 8, 14336)):
    print("product", rows, experts, output, grid("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
        q=P, q_scale=P, w=P, w_scale=P, offsets=P, y=P, rows=rows, experts=experts, hidden=32, output=output)))
for device in (0, 1, 0):
    hip.launches_set_device(device)
    print("tiles", device, grid("mxfp4_grouped_gemm", rr.Mxfp4GroupedGemmArgs(
        q=P, q_scale=P, w=P, w_scale=P, offsets=P, y=P, rows=1 << 20, experts=1, hidden=64, output=256)))
"""


@pytest.mark.skipif(not (ROCM / "include" / "hip").exists(), reason="needs the HIP headers")
def test_grids(tmp_path):
    stand_in = tmp_path / "liblaunches.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                    "-shared", "-fPIC", "-o", str(stand_in), str(REPO / "tests" / "cpp" / "launches.cpp")], check=True)
    out = subprocess.run([sys.executable, "-c", PROGRAM, str(stand_in)], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    most = 2 ** 31 - 1
    want = [
        # workgroups of 512 routes; of 64 routes a token eight tokens; of one token; one a token and one for the offsets
        f"maps {most} 1 256 {-(-most // 512)}", f"maps {most // 64} 64 8 {-(-(most // 64) // 8)}", f"maps {most} 1 1024 {-(-most // 512)}",
        "maps 129 1 8 129", "maps 1 64 8 2",
        "combine 16384", "backward 16384", "gate 16384", "quantize 16384",
        # more workgroups than a launch of the kernel for few rows has, one a compute unit; groups of 16 rows times 64 columns
        f"product {12 * 1024} 1024 {1 << 20} 256", f"product {most} 1 1 256", "product 16 8 14336 1792", "product 16384 8 14336 256",
        "tiles 0 256", "tiles 1 64", "tiles 0 256",
    ]
    assert out.stdout.splitlines() == want
