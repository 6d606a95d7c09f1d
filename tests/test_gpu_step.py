"""Verification steps (Step, appendPacked, attendTree, keep): maps against a
plain walk over the requests, packed appends and kept paths bit for bit
against caches filled by plain appends, tree attention against the formula in
64 bits over what the cache holds."""
from __future__ import annotations

import math
import random

import pytest

from common import log
from test_gpu_dense import D, KINDS, SCALE, _cache, _check, _dt, _fill, _held, _randn

pytestmark = pytest.mark.gpu


def _ints(gpu, values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def _tree(seed, n, absent=0.0):
    """A random tree of n nodes: parents among the last eight nodes, or the cached tokens (-1)."""
    r = random.Random(seed)
    out = []
    for j in range(n):
        p = r.randint(max(-1, j - 8), j - 1) if j else -1
        out.append(r.choice([-2, j, j + 1, 2 ** 31 - 1, -2 ** 31]) if r.random() < absent else p)
    return out


def _paths(parents):
    """Each node's path from the root, itself included; [] where it is absent."""
    out = []
    for j, p in enumerate(parents):
        if p < -1 or p >= j or (p >= 0 and not out[p]):
            out.append([])
        else:
            out.append((out[p] if p >= 0 else []) + [j])
    return out


def _bits(path):
    x = sum(1 << a for a in path)
    return x - (1 << 64) if x >> 63 else x


def _step(gpu, caches, counts, trees, rows=None, most=None, ids=None):
    """A mapped step of these requests (pages reserved for them)."""
    import bsattn
    for c in caches:
        for b, n in zip(ids if ids is not None else range(len(counts)), counts):
            c.reserve(n, seq_ids=[b])
    step = bsattn.Step(caches, rows=rows or max(1, sum(counts)), maxTokens=most or max(1, max(counts)))
    parents = None
    if trees is not None:
        flat = [p for t in trees for p in t]
        parents = _ints(gpu, flat + [7] * (step.rows - len(flat)))
    return step.map(_ints(gpu, counts), parents, seq_ids=ids)


# ---------------------------------------------------------------------------
# maps
# ---------------------------------------------------------------------------
def _check_map(step, lens, counts, trees, ids, fits):
    import torch
    starts, rows = [0], step.rows
    for n in counts:
        starts.append(min(rows, starts[-1] + max(0, n)))
    taken = [max(0, n) if ok else 0 for n, ok in zip(counts, fits)]
    want = {"requests": [-1] * rows, "positions": [0] * rows, "ancestors": [0] * rows,
            "slots": [[-1] * rows for _ in step.caches]}
    for i, n in enumerate(taken):
        paths = _paths(trees[i]) if trees is not None else [list(range(j + 1)) for j in range(n)]
        for j in range(n):
            row = starts[i] + j
            want["requests"][row] = i
            want["positions"][row] = lens[i] + max(0, len(paths[j]) - 1)
            if step.ancestors is not None:
                want["ancestors"][row] = _bits(paths[j])
            for x, c in enumerate(step.caches):
                pages, at = c.seqPages(ids[i]), lens[i] + j
                want["slots"][x][row] = pages[at // c.blockSize] * c.blockSize + at % c.blockSize
    torch.cuda.synchronize()
    assert step.starts.tolist() == starts
    assert step.taken.tolist() == taken
    assert step.ends.tolist() == [[a + n for a, n in zip(lens, taken)]] * len(step.caches)
    for name, w in want.items():
        if name != "ancestors" or step.ancestors is not None:
            assert getattr(step, name).tolist() == w, name


@pytest.mark.parametrize("layers", [1, 3, 7])
@pytest.mark.parametrize("chain", [False, True])
def test_map(gpu, layers, chain):
    """Counts from nothing to 64, lengths in and at the ends of blocks, sequences in another order, rows behind the
    last request, caches of both block sizes with shuffled pages."""
    log(f"[map] layers={layers} chain={chain}")
    lens = [0, 1, 31, 32, 63, 64, 65, 100, 500, 127]
    caches = []
    for x in range(layers):
        c = _cache(lens, 2, 1, 32 if x % 2 else 64, "f16", 4, spare=64)
        _fill(gpu, c, lens, 3 + x)
        caches.append(c)
    ids = [9, 0, 3, 1, 2, 5, 4, 8, 7]
    counts = [64, 1, 0, 33, 2, 17, 64, 5, 0]
    trees = None if chain else [_tree(i, n, 0.2) for i, n in enumerate(counts)]
    for rows in (sum(counts), sum(counts) + 70, sum(counts) + 2000):
        step = _step(gpu, caches, counts, trees, rows=rows, ids=ids)
        _check_map(step, [lens[b] for b in ids], counts, trees, ids, [True] * 9)


def test_map_refuses_requests(gpu):
    """Requests with too many tokens, rows that do not suffice, pages that are missing in one of the caches, counts
    below zero: not taken, and the others are."""
    import bsattn
    log("[map] refused requests")
    lens = [10, 20, 30, 40, 50, 60]
    caches = [_cache(lens, 2, 1, 32, "f16", 4, spare=200) for _ in range(2)]
    for x, c in enumerate(caches):
        _fill(gpu, c, lens, 5 + x)
        c.reserve(100, seq_ids=[0, 1, 2, 3, 4] if x else [0, 1, 2, 3, 4, 5])  # (5: up to 64 in the second one)
    step = bsattn.Step(caches, rows=64, maxTokens=20)
    for counts, fits in (([20, 21, 3, 2, 5, 4], [1, 0, 1, 1, 1, 1]), ([1, 1, 1, 1, 1, 5], [1, 1, 1, 1, 1, 0]),
                         ([20, 20, 20, 5, 4, 1], [1, 1, 1, 0, 0, 0]), ([-3, 4, -2 ** 31, 2, 0, 4], [0, 1, 0, 1, 1, 1]),
                         ([20, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 1, 1], [1, 0, 0, 0, 0, 0])):
        step.map(_ints(gpu, counts))
        _check_map(step, lens, counts, None, range(6), fits)


def test_map_long_chains(gpu):
    """Prompts: chains of thousands of tokens, no ancestors."""
    log("[map] long chains")
    lens, counts = [5, 0, 64], [3000, 1, 2049]
    c = _cache(lens, 2, 1, 64, "f16", 4, spare=3100)
    _fill(gpu, c, lens, 5)
    step = _step(gpu, [c], counts, None, rows=5100)
    assert step.ancestors is None
    _check_map(step, lens, counts, None, range(3), [True] * 3)


# ---------------------------------------------------------------------------
# packed appends
# ---------------------------------------------------------------------------
def _state(c, seqs):
    import torch
    torch.cuda.synchronize()
    out = []
    for s in seqs:
        if c.seqLen(s) == 0:
            out.append([])
            continue
        parts = [t.clone() for part in c.exportQuantized([s]) for t in part] if c.bits else list(c.export([s]))
        out.append(parts + [c.exportSummaries(s)])
    return out


def _same(a, b):
    import torch
    return len(a) == len(b) and all(len(x) == len(y) and all(torch.equal(s, t) for s, t in zip(x, y))
                                    for x, y in zip(a, b))


def _rows(gpu, c, seed, rows, fused=True):
    """Queries, keys and values of packed rows: views into one projection, or dense."""
    dt = {"torch.float16": "f16", "torch.bfloat16": "bf16"}[str(c.dtype)]
    x = _randn(gpu, seed, (rows, c._hq + 2 * c._hkv, D), dt)
    parts = x[:, :c._hq], x[:, c._hq:c._hq + c._hkv], x[:, c._hq + c._hkv:]
    return parts if fused else tuple(p.contiguous() for p in parts)


def _plain_append(c, k, v, b):
    """Rows k, v [n, Hkv, D] appended to sequence b."""
    if k.shape[0]:
        c.append(k.transpose(0, 1)[None].contiguous(), v.transpose(0, 1)[None].contiguous(), seq_ids=[b])


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Tb", [32, 64])
@pytest.mark.parametrize("Hkv", [1, 2, 8])
def test_append_packed(gpu, dtype, bits, Tb, Hkv):
    """Every state and summary is that of plain appends; again with other rows (the first ones are overwritten)."""
    log(f"[append] {dtype} bits={bits} Tb={Tb} Hkv={Hkv}")
    lens = [0, 1, 31, 32, 63, 64, 65, 100, 500, 127]
    counts = [200, 1, 1, 33, 2, 0, 64, 28, 12, 129]
    ids = [1, 0, 2, 3, 9, 5, 4, 8, 7, 6]
    c, ref = (_cache(lens, 2 * Hkv, Hkv, Tb, dtype, bits, spare=260) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, lens, 3)
    step = _step(gpu, [c], counts, None, rows=sum(counts) + 5, ids=ids)
    for seed, fused in ((11, False), (12, True)):
        _, k, v = _rows(gpu, c, seed, step.rows, fused)
        c.appendPacked(k, v, step)
    c.sync()
    for i, b in enumerate(ids):
        a = sum(counts[:i])
        _plain_append(ref, k[a:a + counts[i]], v[a:a + counts[i]], b)
    assert _same(_state(c, range(10)), _state(ref, range(10)))
    # and on by plain appends
    k, v = _randn(gpu, 21, (10, Hkv, 40, D), dtype), _randn(gpu, 22, (10, Hkv, 40, D), dtype)
    c.append(k, v)
    ref.append(k, v)
    assert _same(_state(c, range(10)), _state(ref, range(10)))


# ---------------------------------------------------------------------------
# tree attention
# ---------------------------------------------------------------------------
def _tree_reference(c, q, step, lens, counts, trees, ids=None, window=None, sinks=None, scale=SCALE):
    """[rows, Hq, D] in 64 bits (zeros behind the last request) and the rows that are somebody's."""
    import torch
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    G, first = c._hq // c._hkv, 0
    for i, (P, N) in enumerate(zip(lens, counts)):
        if N == 0:
            continue
        k, v = _held(c, ids[i] if ids is not None else i)
        paths = _paths(trees[i]) if trees is not None else [list(range(j + 1)) for j in range(N)]
        see = torch.zeros((N, P + N), dtype=torch.bool)
        for j, path in enumerate(paths):
            if not path:
                continue
            pos = P + len(path) - 1
            see[j, (max(0, pos - window + 1) if window else 0):P] = True
            see[j, [P + a for d, a in enumerate(path) if not window or P + d > pos - window]] = True
        hide = ~see.to(q.device)[:, None]
        for h in range(c._hkv):
            heads = slice(h * G, (h + 1) * G)
            x = q[first:first + N, heads].double()
            # (what a node does not see may be anything)
            for j in range(N):
                on = see[j].to(q.device)
                if not on.any():
                    continue
                s = x[j] @ k[h][on].t() * scale
                top = s.amax(-1, keepdim=True)
                if sinks is not None:
                    sk = sinks[heads].double()[:, None]
                    top = torch.maximum(top, sk)
                p = torch.exp(s - top)
                total = p.sum(-1, keepdim=True)
                if sinks is not None:
                    total = total + torch.exp(sk - top)
                out[first + j, heads] = p @ v[h][on] / total
        del hide
        first += N
    return out


def _verify(gpu, c, lens, counts, trees, seed, what="", ids=None, window=None, sinks=None, rows=None, fused=True,
            mangle=None):
    """Appends a step's rows, attends and checks; the step."""
    import torch
    step = _step(gpu, [c], counts, trees, rows=rows, ids=ids)
    q, k, v = _rows(gpu, c, seed, step.rows, fused)
    if mangle is not None:
        mangle(q, k, v)
    c.appendPacked(k, v, step)
    out = torch.full((step.rows, c._hq, D), 7.0, dtype=c.dtype, device=gpu)
    c.attendTree(q, step, SCALE, window=window, sinks=sinks, out=out)
    c.sync()
    want = _tree_reference(c, q, step, lens, counts, trees, ids, window, sinks)
    n = sum(counts)
    assert (out[n:] == 7).all()
    dt = {"torch.float16": "f16", "torch.bfloat16": "bf16"}[str(c.dtype)]
    if n:
        _check(out[:n, :, None], want[:n], dt, what)
    if trees is not None:
        gone = [sum(counts[:i]) + j for i, t in enumerate(trees) for j, p in enumerate(_paths(t)) if not p]
        assert (out[gone] == 0).all()
    return step


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (4, 2), (32, 8), (16, 2), (64, 4), (16, 1)])
@pytest.mark.parametrize("Tb", [32, 64])
def test_tree(gpu, dtype, bits, Hq, Hkv, Tb):
    """Lengths from nothing to many parts, trees from one node to 64, ends inside units and pages."""
    log(f"[tree] {dtype} bits={bits} {Hq}/{Hkv} Tb={Tb}")
    lens = [1, 0, 31, 32, 33, 64, 65, 500, 1000, 2049, 0, 127]
    counts = [1, 5, 2, 64, 17, 0, 31, 33, 63, 8, 1, 12]
    c = _cache(lens, Hq, Hkv, Tb, dtype, bits, spare=64)
    _fill(gpu, c, lens, 100 + Hq + Tb, salient=True)
    _verify(gpu, c, lens, counts, [_tree(i, n) for i, n in enumerate(counts)], 7, rows=sum(counts) + 3)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("most", [1, 3, 4, 8, 16, 64])
def test_tree_sizes(gpu, dtype, bits, most):
    """Every number of column tiles, with chains; one long sequence, split over the GPU."""
    log(f"[tree sizes] {dtype} bits={bits} {most}")
    lens, counts = [9000, 77], [most, max(1, most - 1)]
    c = _cache(lens, 8, 2, 64, dtype, bits, spare=64)
    _fill(gpu, c, lens, 5)
    _verify(gpu, c, lens, counts, None, 9)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("window", [1, 2, 7, 33, 64, 100, 1000, 100000])
def test_tree_windows(gpu, dtype, bits, window):
    """Windows from the node alone to more than there is; sinks beside them; absent nodes; sequences in another order."""
    log(f"[tree windows] {dtype} bits={bits} {window}")
    lens, counts, ids = [700, 3, 64, 2100], [40, 64, 9, 25], [2, 0, 3, 1]
    c = _cache([lens[ids.index(b)] for b in range(4)], 8, 2, 32, dtype, bits, spare=64)
    _fill(gpu, c, [lens[ids.index(b)] for b in range(4)], 5)
    sinks = _randn(gpu, 3, (8,), "f16").float() + 2
    sinks[3] = -math.inf
    _verify(gpu, c, lens, counts, [_tree(i, n, 0.1) for i, n in enumerate(counts)], 9, window=window, sinks=sinks,
            ids=ids)


@pytest.mark.parametrize("dtype,bits", [("f16", 0), ("bf16", 0)])
@pytest.mark.parametrize("window", [None, 20])
def test_unseen_values(gpu, dtype, bits, window):
    """Infinities and NaN in keys and values that a node does not see change nothing of its output: siblings', those
    of rejected rows in the same pages, those before the window."""
    import torch
    log(f"[tree unseen] {dtype} window={window}")
    lens, N = [100], 33
    c, clean = (_cache(lens, 8, 2, 64, dtype, bits, spare=64) for _ in range(2))
    for x in (c, clean):
        _fill(gpu, x, lens, 5)
    # a path of even nodes, one of odd ones; the odd ones' keys and values are anything
    tree = [[-1, -1] + list(range(0, N - 2))]
    out = []
    for x, bad in ((clean, False), (c, True)):
        step = _step(gpu, [x], [N], tree)
        q, k, v = _rows(gpu, x, 8, N, fused=False)
        if bad:
            # (rows of an earlier step in the same places)
            x.appendPacked(torch.full_like(k, math.nan), torch.full_like(v, math.inf), step)
            k[1::2] = math.nan
            v[1::2, :, ::3] = math.inf
            v[3::2, :, 1::3] = -math.inf
            v[5::2, :, 2::5] = math.nan
        x.appendPacked(k, v, step)
        out.append(x.attendTree(q, step, SCALE, window=window))
    torch.cuda.synchronize()
    assert torch.equal(out[0][0::2], out[1][0::2])
    assert not torch.isfinite(out[1][1::2]).all()


def test_attended_infinities(gpu):
    """An infinite value that a node does see is infinite or NaN in its dim, and there alone."""
    import torch
    log("[tree infinite]")
    for dtype in ("f16", "bf16"):
        c = _cache([100], 8, 2, 64, dtype, spare=64)
        _fill(gpu, c, [100], 5)
        step = _step(gpu, [c], [4], [[-1, 0, 0, 1]])
        q, k, v = _rows(gpu, c, 8, 4, fused=False)
        base = None
        for bad in (False, True):
            if bad:
                v[1, :, 5] = math.inf
            c.appendPacked(k, v, step)
            out = c.attendTree(q, step, SCALE)
            if base is None:
                base = out
        torch.cuda.synchronize()
        assert torch.equal(out[[0, 2]], base[[0, 2]])
        for row in (1, 3):
            assert not torch.isfinite(out[row, :, 5]).any()
            rest = [d for d in range(D) if d != 5]
            assert torch.equal(out[row][:, rest], base[row][:, rest])


def test_nan_queries(gpu):
    """A query of NaN gives NaN in its own row alone; an absent node's gives zeros."""
    import torch
    log("[tree NaN]")
    for T in (50, 9000):
        c = _cache([T], 8, 2, 64, "bf16", spare=64)
        _fill(gpu, c, [T], 5)
        step = _step(gpu, [c], [4], [[-1, 0, -2, 0]])
        q, k, v = _rows(gpu, c, 8, 4, fused=False)
        c.appendPacked(k, v, step)
        base = c.attendTree(q, step, SCALE)
        q[1:3] = math.nan
        out = c.attendTree(q, step, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(out[[0, 3]], base[[0, 3]])
        assert torch.isnan(out[1]).all() and (out[2] == 0).all()


# ---------------------------------------------------------------------------
# kept paths
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Tb", [32, 64])
def test_keep(gpu, dtype, bits, Tb):
    """States and summaries are those of caches that were given the kept tokens alone; then nothing is kept."""
    import torch
    log(f"[keep] {dtype} bits={bits} Tb={Tb}")
    lens = [0, 1, 5, 31, 32, 63, 64, 100, 500, 127, 60]
    counts = [64, 1, 17, 33, 2, 64, 0, 28, 12, 64, 9]
    kept = [list(range(64)), [0], [0, 1, 2, 3], [0, 2, 5, 8, 13, 31, 32], [1], list(range(1, 64, 2)), [], [],
            [3, 11], list(range(20, 64)), [0, 1, 2, 3, 8]]
    B, Hkv = len(lens), 2
    c, ref = (_cache(lens, 8, Hkv, Tb, dtype, bits, spare=100) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, lens, 3)
    before = _state(c, range(B))
    step = _step(gpu, [c], counts, None)
    _, k, v = _rows(gpu, c, 12, step.rows)
    lists = _ints(gpu, [x + [0] * (64 - len(x)) for x in kept])
    c.appendPacked(k, v, step)
    c.keep(step, lists, _ints(gpu, [len(x) for x in kept]))
    for i in range(B):
        a = sum(counts[:i])
        at = torch.tensor([a + j for j in kept[i]], dtype=torch.long, device=gpu)
        _plain_append(ref, k[at], v[at], i)
    c.sync()
    assert [c.seqLen(b) for b in range(B)] == [n + len(x) for n, x in zip(lens, kept)]
    assert _same(_state(c, range(B)), _state(ref, range(B)))
    # and on by plain appends (the host's own view again)
    more = [_randn(gpu, 21 + x, (B, Hkv, 33, D), dtype) for x in (0, 1)]
    c.append(*more)
    ref.append(*more)
    assert _same(_state(c, range(B)), _state(ref, range(B)))
    # all of it taken back
    c.trim(33)
    for b in range(B):
        c.trim(len(kept[b]), seq_ids=[b])
    step = _step(gpu, [c], counts, None)
    c.appendPacked(k, v, step)
    c.keep(step, lists, _ints(gpu, [len(x) for x in kept]))
    c.keep(step, lists, _ints(gpu, [0] * B))
    c.sync()
    assert _same(_state(c, range(B)), before)


def test_keep_lists_end(gpu):
    """A list ends at the first entry that does not ascend or is no node; counts past the width or below zero."""
    import torch
    log("[keep] lists")
    lens = [40] * 6
    c, ref = (_cache(lens, 8, 2, 32, "bf16", spare=40) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, lens, 3)
    step = _step(gpu, [c], [8] * 6, None)
    _, k, v = _rows(gpu, c, 12, step.rows)
    c.appendPacked(k, v, step)
    lists = [[1, 3, 3, 4], [5, 4, 6, 7], [0, 8, 1, 2], [-1, 1, 2, 3], [2, 3, 4, 5], [0, 1, 2, 3]]
    c.keep(step, _ints(gpu, lists), _ints(gpu, [4, 4, 4, 4, 2 ** 31 - 1, -5]))
    want = [[1, 3], [5], [0], [], [2, 3, 4, 5], []]
    for i, path in enumerate(want):
        at = torch.tensor([8 * i + j for j in path], dtype=torch.long, device=gpu)
        _plain_append(ref, k[at], v[at], i)
    c.sync()
    assert [c.seqLen(b) for b in range(6)] == [40 + len(x) for x in want]
    assert _same(_state(c, range(6)), _state(ref, range(6)))
