"""Kernels that calls launch, seen by a stand-in for HIP in a process of its own (no GPU is used:
tests/cpp/kernels.cpp, tests/cpp/launches.cpp)."""
from __future__ import annotations

import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
ROCM = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
P = 4096  # a pointer that is never followed

PROGRAM = """
import ctypes, json, sys
names = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
ctypes.CDLL(sys.argv[2], mode=ctypes.RTLD_GLOBAL)
names.kernels_launched.restype = names.kernels_registered.restype = ctypes.c_char_p
import raggedroute_amd as rr
from raggedroute_amd import _capi
arguments = dict(_capi._OP_ENTRIES)
out = []
for entry, fields in json.load(sys.stdin):
    if "kernel" in fields:
        fields["kernel"] = rr.kernel(rr.KernelFamily(fields["kernel"]))
    args = arguments[entry](**fields)
    size = getattr(rr, f"get_{entry}_workspace_size")(args)
    status = getattr(rr, entry)(args, rr.RuntimeContext(architecture=int(rr.DeviceArchitecture.kGfx950), workspace=4096,
                                                        workspace_bytes=size))
    assert status.ok(), (entry, fields, status.message)
    out.append(names.kernels_launched().decode().split())
json.dump([out, [n for n in names.kernels_registered().decode().split() if "2rr4kern" in n]], sys.stdout)
"""


def launched(folder, calls):
    """Mangled names of the kernels that every (entry, fields) launches, and of all that the library has."""
    if not (ROCM / "include" / "hip").exists():
        pytest.skip("needs the HIP headers")
    for name in ("kernels", "launches"):
        subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                        "-shared", "-fPIC", "-o", str(folder / f"lib{name}.so"), str(REPO / "tests" / "cpp" / f"{name}.cpp")],
                       check=True)
    out = subprocess.run([sys.executable, "-c", PROGRAM, str(folder / "libkernels.so"), str(folder / "liblaunches.so")],
                         cwd=REPO, input=json.dumps(calls), capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return json.loads(out.stdout)
