"""Verification steps' host side on the CPU: refusals, the order of the calls,
workspaces, and the cut of a tree attention into parts (tests/capi_host)."""
from __future__ import annotations

import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "mlx-swift-lm_amd", "csrc")
ROCM = os.environ.get("ROCM", "/opt/rocm")


@pytest.mark.parametrize("program,sources,stubs", [
    ("tree_parts", ["bsattn_tree_plan.cpp"], []),
    ("steps", ["bsattn_capi.cpp", "bsattn_ops.cpp", "bsattn_steps.cpp", "bsattn_tree_plan.cpp"],
     ["stubs.cpp", "stubs_ops.cpp"])])
def test_steps(tmp_path, program, sources, stubs):
    exe = str(tmp_path / program)
    host = os.path.join(HERE, "capi_host")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-D_GLIBCXX_ASSERTIONS", "-D__HIP_PLATFORM_AMD__",
                    "-Xlinker", "--no-undefined", f"-I{ROCM}/include", *(os.path.join(CSRC, f) for f in sources),
                    *(os.path.join(host, f) for f in (*stubs, program + ".cpp")), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
