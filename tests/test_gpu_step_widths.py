"""Tree attention by every width of its waves, for every type of cache: 16 to
256 columns a workgroup, those of 64 and 128 in waves of one column tile (few
units a workgroup) and of two (many)."""
from __future__ import annotations

import math

import pytest

from common import log
from test_gpu_dense import KINDS, _cache, _fill, _randn
from test_gpu_step import _tree, _verify

pytestmark = pytest.mark.gpu

# (Hq, Hkv, tokens per block, cached tokens, drafts, window, column tiles of a workgroup, whether its waves hold one)
SHAPES = [
    (32, 8, 64, [3000], [4], None, 1, False),
    (32, 8, 64, [3000, 70], [7, 3], None, 2, False),
    (32, 8, 64, [3000, 70], [16, 9], None, 4, True),
    (32, 8, 32, [20000], [16], None, 4, False),
    (32, 8, 64, [20003], [13], None, 4, False),
    (32, 8, 64, [21000, 333], [9, 15], 17000, 4, False),
    (32, 8, 64, [3000, 70], [32, 17], None, 8, True),
    (32, 8, 64, [20000], [32], None, 8, False),
    (32, 8, 32, [19999], [25], None, 8, False),
    (32, 8, 64, [21000, 64], [27, 31], 17000, 8, False),
    (16, 1, 64, [3000], [16], None, 16, False),
    (32, 4, 32, [20000, 1], [33, 64], 16500, 16, False),
]


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_widths(gpu, dtype, bits, shape):
    Hq, Hkv, Tb, lens, counts, window = shape[:6]
    log(f"[widths] {dtype} bits={bits} {shape}")
    c = _cache(lens, Hq, Hkv, Tb, dtype, bits, spare=64)
    _fill(gpu, c, lens, 5, salient=True)
    sinks = None
    if window:
        sinks = _randn(gpu, 3, (Hq,), "f16").float() + 2
        sinks[3] = -math.inf
    _verify(gpu, c, lens, counts, [_tree(i, n, 0.1) for i, n in enumerate(counts)], 9, window=window, sinks=sinks)
