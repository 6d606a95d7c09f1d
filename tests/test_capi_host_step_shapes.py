"""The shapes of test_gpu_step_widths.py and test_gpu_step_bits.py reach every
tree attention kernel: every number of column tiles a workgroup, in waves of
one and of two (tests/capi_host/tree_shapes.cpp)."""
from __future__ import annotations

import os
import subprocess

import test_gpu_step_bits as bits
import test_gpu_step_widths as widths

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "mlx-swift-lm_amd", "csrc")
HOST = os.path.join(HERE, "capi_host")
ROCM = os.environ.get("ROCM", "/opt/rocm")
EVERY = {(1, False), (2, False), (4, True), (4, False), (8, True), (8, False), (16, False)}


def test_shapes_reach_every_width(tmp_path):
    exe = str(tmp_path / "tree_shapes")
    sources = ["bsattn_capi.cpp", "bsattn_ops.cpp", "bsattn_steps.cpp", "bsattn_tree_plan.cpp"]
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-D_GLIBCXX_ASSERTIONS", "-D__HIP_PLATFORM_AMD__",
                    "-Xlinker", "--no-undefined", f"-I{ROCM}/include", *(os.path.join(CSRC, f) for f in sources),
                    *(os.path.join(HOST, f) for f in ("stubs.cpp", "stubs_ops.cpp", "tree_shapes.cpp")), "-o", exe],
                   check=True)
    shapes = [s[:6] for s in widths.SHAPES] + [(Hq, Hkv, 64, [T], [N], None) for Hq, Hkv, T, N in bits.WIDTHS]
    calls = "\n".join(" ".join(str(x) for x in (Hq, Hkv, Tb, max(counts), window or 0, len(lens), *lens))
                      for Hq, Hkv, Tb, lens, counts, window in shapes)
    r = subprocess.run([exe], input=calls, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    got = [(int(a), b == "1") for a, b in (line.split() for line in r.stdout.splitlines())]
    assert len(got) == len(shapes)
    assert got[:len(widths.SHAPES)] == [s[6:] for s in widths.SHAPES]
    assert set(got[:len(widths.SHAPES)]) == EVERY and set(got[len(widths.SHAPES):]) == EVERY
