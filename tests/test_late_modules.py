"""Which code objects a context loads, and when (CPU only): the library's host
sources with a HIP runtime that counts instead of loading
(tests/fuzz/late_modules.cpp). A context that never touches the key/value cache
loads none of the attention's kernels; the first one on a device that does loads
those of its head size, for all, whatever threads or captures the call comes from."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.parametrize("sanitize", ["address,undefined", "thread"])
def test_the_attention_is_loaded_at_its_first_use(tmp_path, sanitize):
    gxx = shutil.which("g++")
    if not gxx or not os.path.exists(os.path.join(ROCM, "include", "hip", "hip_runtime_api.h")):
        pytest.skip("needs g++ and the HIP headers")
    exe = str(tmp_path / "late_modules")
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-pthread", "-D__HIP_PLATFORM_AMD__", f"-fsanitize={sanitize}", f"-I{ROOT}/include",
           f"-I{ROOT}/vortx_amd/csrc", f"-I{ROCM}/include", f"{ROOT}/tests/fuzz/late_modules.cpp",
           *[f"{ROOT}/vortx_amd/csrc/{s}" for s in ("vx_host.cpp", "vx_attn.cpp", "vx_layout.cpp")], "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0 and "cannot find" in r.stderr and "san" in r.stderr:
        pytest.skip("sanitizer runtime not installed")
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fine" in r.stdout, (r.stdout + r.stderr)[-3000:]
