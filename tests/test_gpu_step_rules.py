"""Verification steps beside other calls: requests prefilled while a step is
under way, and captured steps mapped for other requests."""
from __future__ import annotations

import pytest

from common import log
from test_gpu_dense import KINDS, SCALE, _cache, _fill, _randn
from test_gpu_step import _ints, _paths, _plain_append, _rows, _same, _state, _step, _tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", KINDS)
def test_prompt_beside_a_step(gpu, dtype, bits):
    """A request is prefilled, another one trimmed and a third let go between a step's attention and its kept paths:
    the attention gives the same bits, and the states are those of a cache that was given the kept tokens."""
    import bsattn
    import torch
    log(f"[beside] {dtype} bits={bits}")
    lens, ids, counts = [150, 70, 0, 90, 64], [3, 0], [20, 33]
    c, ref = (_cache([200] * 5, 8, 2, 64, dtype, bits, spare=64) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, lens, 3)
    trees = [_tree(i, n) for i, n in enumerate(counts)]
    step = _step(gpu, [c], counts, trees, ids=ids)
    q, k, v = _rows(gpu, c, 11, step.rows)
    c.appendPacked(k, v, step)
    first = c.attendTree(q, step, SCALE)
    c.sync()
    prompt = [_randn(gpu, 50 + x, (1, 2, 130, 128), "f16" if bits else dtype) for x in (0, 1)]
    for x in (c, ref):
        x.append(*prompt, seq_ids=[2])
        x.trim(10, seq_ids=[1])
        x.reset([4])
    assert torch.equal(c.attendTree(q, step, SCALE), first)
    kept = [max(_paths(t), key=len) for t in trees]
    c.keep(step, _ints(gpu, [p + [0] * (33 - len(p)) for p in kept]), _ints(gpu, [len(p) for p in kept]))
    c.sync()
    for i, b in enumerate(ids):
        at = torch.tensor([sum(counts[:i]) + j for j in kept[i]], dtype=torch.long, device=gpu)
        _plain_append(ref, k[at], v[at], b)
    assert _same(_state(c, range(5)), _state(ref, range(5)))
    c.trim(1, seq_ids=[0])
    with pytest.raises(bsattn.BsattnError, match="changed"):
        c.keep(step, _ints(gpu, [[0], [0]]), _ints(gpu, [0, 0]))


def test_captured_step_for_other_requests(gpu):
    """A captured step, then mapped for one request less: its eager calls are refused; mapped as it was captured they
    are taken, with the lengths of a cache that was given the kept tokens."""
    import bsattn
    import torch
    log("[other requests]")
    N = 4
    a, b = (_cache([40, 70], 4, 2, 32, "f16", spare=64) for _ in range(2))  # (two layers: the second's ends lie behind n of the first)
    for x in (a, b):
        _fill(gpu, x, [40, 70], 3)
        x.reserve(40)
    step = bsattn.Step([a, b], rows=2 * N, maxTokens=N)
    counts, kept, many = _ints(gpu, [3, 4]), _ints(gpu, [[0, 1]] * 2), _ints(gpu, [2, 1])
    _, k, v = _rows(gpu, a, 1, 2 * N, fused=False)

    def first():
        step.map(counts)
        for c in (a, b):
            c.appendPacked(k, v, step)

    first()
    for c in (a, b):
        c.keep(step, kept, _ints(gpu, [0, 0]))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        first()
    for turn in range(3):
        step.map(_ints(gpu, [2]), seq_ids=[1])
        g.replay()
        torch.cuda.synchronize()
        for c in (a, b):
            with pytest.raises(bsattn.BsattnError, match="captured for other requests"):
                c.keep(step, kept[:1], many[:1])
        step.map(counts)  # (over the drafts that the replay appended: they are kept with it)
        for c in (a, b):
            c.appendPacked(k, v, step)
            c.keep(step, kept, many)
            c.sync()
        want = [40 + 5 * (turn + 1), 70 + 5 * (turn + 1)]
        assert [[c.seqLen(i) for i in (0, 1)] for c in (a, b)] == [want, want]
