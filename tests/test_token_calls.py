"""The C++ calls of the token and 4-bit operators, compiled against the headers alone (tests/cpp/token_calls.cpp)."""
from __future__ import annotations

import subprocess

import pytest

from stand_in import REPO, ROCM


@pytest.mark.skipif(not (ROCM / "include" / "hip").exists(), reason="needs the HIP headers")
def test_calls_reach_the_c_entries(tmp_path):
    program = tmp_path / "token_calls"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", f"-I{REPO / 'include'}",
                    f"-I{ROCM}/include", str(REPO / "tests" / "cpp" / "token_calls.cpp"), "-o", str(program)], check=True)
    out = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout == "token calls OK\n", out.stdout + out.stderr
