"""Grids of the expert block's persistent kernels, by launches that a stand-in for HIP counts
(no GPU is used: tests/cpp/launches.cpp)."""
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
args = rr.GatedFfnArgs(x=P, w_gate=P, w_up=P, w_down=P, offsets=P, act=P, y=P, rows=1 << 20, experts=1, hidden=64,
                       inner=256, output=256)
context = rr.RuntimeContext(architecture=int(rr.DeviceArchitecture.kGfx950))
for device in (0, 1, 0):
    hip.launches_set_device(device)
    assert rr.gated_ffn(args, context).ok()
    print(hip.launches_grid())
"""


@pytest.mark.skipif(not (ROCM / "include" / "hip").exists(), reason="needs the HIP headers")
def test_grids_follow_the_current_device(tmp_path):
    """One workgroup a compute unit of the device that the call runs on, whichever was first."""
    stand_in = tmp_path / "liblaunches.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                    "-shared", "-fPIC", "-o", str(stand_in), str(REPO / "tests" / "cpp" / "launches.cpp")], check=True)
    out = subprocess.run([sys.executable, "-c", PROGRAM, str(stand_in)], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == ["256", "64", "256"]
