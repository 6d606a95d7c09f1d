"""Which calls with a verification step the host takes and which it refuses,
around captures and other sequences' calls (tests/capi_host/step_rules.cpp)."""
from __future__ import annotations

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "mlx-swift-lm_amd", "csrc")
HOST = os.path.join(HERE, "capi_host")
ROCM = os.environ.get("ROCM", "/opt/rocm")


def test_step_rules(tmp_path):
    exe = str(tmp_path / "step_rules")
    sources = ["bsattn_capi.cpp", "bsattn_ops.cpp", "bsattn_steps.cpp", "bsattn_tree_plan.cpp"]
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-D_GLIBCXX_ASSERTIONS", "-D__HIP_PLATFORM_AMD__",
                    "-Xlinker", "--no-undefined", f"-I{ROCM}/include", *(os.path.join(CSRC, f) for f in sources),
                    *(os.path.join(HOST, f) for f in ("stubs.cpp", "stubs_ops.cpp", "step_rules.cpp")), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
