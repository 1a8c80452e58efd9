"""No kernel of the cache and its attention is left without a call, on the CPU (tests/fuzz/attn_reach.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


def test_every_kernel_is_reached(tmp_path):
    gxx = shutil.which("g++")
    if not gxx or not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")):
        pytest.skip("needs g++ and the HIP headers")
    exe = str(tmp_path / "attn_reach")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include", f"-I{ROOT}/vortx_amd/csrc",
                        f"-I{ROCM}/include", f"{ROOT}/tests/fuzz/attn_reach.cpp",
                        *[f"{ROOT}/vortx_amd/csrc/{s}" for s in ("vx_host.cpp", "vx_attn.cpp", "vx_layout.cpp")], "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fine" in r.stdout, (r.stdout + r.stderr)[-3000:]
