"""Rotation of very many heads, on the CPU (tests/fuzz/step_limits.cpp)."""
import os
import shutil
import subprocess

import pytest

from tests.test_step_host import ROCM, ROOT


def test_limits(tmp_path):
    gxx = shutil.which("g++")
    if not gxx or not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")):
        pytest.skip("needs g++ and the HIP headers")
    exe = str(tmp_path / "step_limits")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include", f"-I{ROOT}/vortx_amd/csrc",
                        f"-I{ROCM}/include", f"{ROOT}/tests/fuzz/step_limits.cpp",
                        *[f"{ROOT}/vortx_amd/csrc/{s}" for s in ("vx_host.cpp", "vx_attn.cpp", "vx_layout.cpp")], "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fine" in r.stdout, (r.stdout + r.stderr)[-3000:]
