"""The units, parts and partials of tree attentions by the kernels' own integer
code (tests/capi_host/tree_units.cpp)."""
from __future__ import annotations

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "mlx-swift-lm_amd", "csrc")
ROCM = os.environ.get("ROCM", "/opt/rocm")


def test_tree_units(tmp_path):
    exe = str(tmp_path / "tree_units")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-D_GLIBCXX_ASSERTIONS", "-D__HIP_PLATFORM_AMD__",
                    "-Xlinker", "--no-undefined", f"-I{ROCM}/include", os.path.join(CSRC, "bsattn_tree_plan.cpp"),
                    os.path.join(HERE, "capi_host", "tree_units.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
