"""Which kernel a 4-bit product takes, by the launches that a stand-in for HIP sees (no GPU is used:
tests/cpp/kernels.cpp, tests/cpp/launches.cpp). The tests on the GPU take their cases from the same lists, so that
a rule that sends them elsewhere fails here."""
from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))

PROGRAM = """
import ctypes, json, re, sys
names = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
ctypes.CDLL(sys.argv[2], mode=ctypes.RTLD_GLOBAL)
names.kernels_launched.restype = ctypes.c_char_p
import raggedroute_amd as rr
P = 4096
CODES = dict(f32=int(rr.ScalarType.kFp32), f16=int(rr.ScalarType.kFp16), bf16=int(rr.ScalarType.kBf16))
context = rr.RuntimeContext(architecture=int(rr.DeviceArchitecture.kGfx950))
out = []
for rows, experts, k, n, dtype, gated in json.load(sys.stdin):
    up = dict(w_up=P, w_up_scale=P) if gated else {}
    status = rr.mxfp4_grouped_gemm(rr.Mxfp4GroupedGemmArgs(
        q=P, q_scale=P, w=P, w_scale=P, offsets=P, y=P, rows=rows, experts=experts, hidden=k, output=n, dtype=CODES[dtype],
        **up), context)
    assert status.ok(), status.message
    launched = names.kernels_launched().decode().split()
    assert len(launched) == 1, launched
    name = launched[0]
    tile = re.search(r"rr_mxfp4_gemm_kernel.*Li(\\d+)E", name)
    few = re.search(r"rr_mxfp4_rows_kernel.*Li(\\d+)ELi(\\d+)ELb(\\d)E", name)
    out.append([int(tile[1])] if tile else [int(v) for v in few.groups()])
json.dump(out, sys.stdout)
"""

pytestmark = pytest.mark.skipif(not (ROCM / "include" / "hip").exists(), reason="needs the HIP headers")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Rows of a tile, or waves, weight rows and `past the caches` of the kernel for few rows, of every call."""
    folder = tmp_path_factory.mktemp("stand_in")
    for name in ("kernels", "launches"):
        subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                        "-shared", "-fPIC", "-o", str(folder / f"lib{name}.so"), str(REPO / "tests" / "cpp" / f"{name}.cpp")],
                       check=True)

    def run(calls):
        out = subprocess.run([sys.executable, "-c", PROGRAM, str(folder / "libkernels.so"), str(folder / "liblaunches.so")],
                             cwd=REPO, input=json.dumps(calls), capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out.stderr
        return json.loads(out.stdout)

    return run


def test_tiles(kernels):
    from mxfp4_cases import FORMS, TILES
    calls, want = [], []
    for counts, k, n, tile in TILES:
        for dtype, gated, _ in FORMS:
            calls.append([sum(counts) + 2, len(counts), k, n, dtype, gated])
            want.append([tile])
    got = kernels(calls)
    assert not [(c, g, w) for c, g, w in zip(calls, got, want) if g != w]


def test_tiles_of_special_cases(kernels):
    from mxfp4_cases import TILE_SIZES
    from test_gpu_block_offsets import OFFSETS
    calls, want = [], []
    for tile, (rows, n) in TILE_SIZES.items():
        experts = [len(o) - 1 for o in OFFSETS.values()] + [4]
        calls += [[e * rows, e, 320, n, dtype, gated] for e in experts for dtype in ("f32", "bf16") for gated in (False, True)]
        want += [[tile]] * (4 * len(experts))
    assert kernels(calls) == want
