"""The operators' host side (forks' page bookkeeping, refusals, workspaces) on
the CPU: bsattn_capi.cpp and bsattn_ops.cpp linked with a stub HIP runtime and
stub launchers (tests/capi_host)."""
from __future__ import annotations

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "mlx-swift-lm_amd", "csrc")
ROCM = os.environ.get("ROCM", "/opt/rocm")


def test_forks_and_refusals(tmp_path):
    exe = str(tmp_path / "forks")
    host = os.path.join(HERE, "capi_host")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-D_GLIBCXX_ASSERTIONS", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                    os.path.join(CSRC, "bsattn_capi.cpp"), os.path.join(CSRC, "bsattn_ops.cpp"),
                    *(os.path.join(host, f) for f in ("stubs.cpp", "stubs_ops.cpp", "forks.cpp")), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
