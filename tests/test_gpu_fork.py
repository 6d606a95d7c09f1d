"""Forks (bsattn_fork): branches of a prompt share its full pages, decode and
export as caches of their own would, and give their pages back; and the
operators together as a decoding program runs them."""
from __future__ import annotations

import pytest

from common import log
from test_gpu_dense import D, KINDS, SCALE, _cache, _check, _dt, _fill, _randn, _reference

pytestmark = pytest.mark.gpu


def _state(c, seqs):
    import torch
    torch.cuda.synchronize()
    out = []
    for s in seqs:
        if c.seqLen(s) == 0:
            out.append([])
        elif c.bits:
            out.append([t.clone() for part in c.exportQuantized([s]) for t in part])
        else:
            out.append(list(c.export([s])))
        out[-1] = out[-1] + [c.exportSummaries(s)]
    return out


def _same(a, b):
    import torch
    return len(a) == len(b) and all(len(x) == len(y) and all(torch.equal(s, t) for s, t in zip(x, y))
                                    for x, y in zip(a, b))


def _tokens(gpu, c, seed, n, L=1):
    dt = "f16" if c.bits else {"torch.float16": "f16", "torch.bfloat16": "bf16"}[str(c.dtype)]
    return (_randn(gpu, seed, (n, c._hkv, L, D), dt), _randn(gpu, seed + 1, (n, c._hkv, L, D), dt))


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Tb", [32, 64])
@pytest.mark.parametrize("T", [1, 31, 64, 100, 640, 1999])
def test_branches(gpu, dtype, bits, Tb, T):
    """Branches and their prompt go on by themselves: every state and output is
    that of caches filled token by token."""
    import torch
    log(f"[fork] {dtype} bits={bits} Tb={Tb} T={T}")
    c = _cache([T, 0, 0, 0, 0], 8, 2, Tb, dtype, bits, spare=80)
    ref = _cache([T, 0, 0, 0, 0], 8, 2, Tb, dtype, bits, spare=80)
    for x in (c, ref):
        x.shuffleFreePages(3)
    free = c.freePages
    k, v = _tokens(gpu, c, 1, 1, T)
    for b in range(4):
        ref.append(k, v, seq_ids=[b])
    c.append(k, v, seq_ids=[0])
    held = free - c.freePages
    c.fork([0, 0, 0], [1, 2, 3])
    assert free - c.freePages == held + (3 if T % Tb else 0)
    assert [c.seqPages(b)[:T // Tb] for b in (1, 2, 3)] == [c.seqPages(0)[:T // Tb]] * 3
    assert _same(_state(c, range(5)), _state(ref, range(5)))
    # each goes on: one token, then many, on the prompt as on its branches
    for step, L in enumerate((1, 3, 70)):
        k, v = _tokens(gpu, c, 10 + step, 4, L)
        c.append(k, v)
        ref.append(k, v)
        assert _same(_state(c, range(4)), _state(ref, range(4))), f"step {step}"
    q = _randn(gpu, 8, (4, 8, 1, D), dtype)
    assert torch.equal(c.decode(q, SCALE), ref.decode(q, SCALE))
    _check(c.decodeDense(q, SCALE), _reference(ref, q), dtype)
    # and away
    c.reset([0, 2])
    ref.reset([0, 2])
    assert _same(_state(c, range(4)), _state(ref, range(4)))
    c.reset([1, 3])
    assert c.freePages == free


@pytest.mark.parametrize("dtype,bits", KINDS)
def test_trim_into_shared_blocks(gpu, dtype, bits):
    """Trims that end inside shared blocks take copies; nobody else's tokens
    change, whoever goes first, and the last holder keeps the page."""
    T = 300
    for order in ([0, 1, 2], [2, 0, 1], [1]):
        c = _cache([T, 0, 0], 8, 2, 64, dtype, bits)
        ref = _cache([T, 0, 0], 8, 2, 64, dtype, bits)
        k, v = _tokens(gpu, c, 1, 1, T)
        for b in range(3):
            ref.append(k, v, seq_ids=[b])
        free = c.freePages
        c.append(k, v, seq_ids=[0])
        c.fork([0, 0], [1, 2])
        for n, L in ((200, 30), (64, 1), (1, 150), (10, 5)):
            for s in order:
                assert c.trim(n, seq_ids=[s]) == ref.trim(n, seq_ids=[s])
                assert _same(_state(c, range(3)), _state(ref, range(3))), (order, n, s)
                x, y = _tokens(gpu, c, 50 + s, 1, L)
                c.append(x, y, seq_ids=[s])
                ref.append(x, y, seq_ids=[s])
                assert _same(_state(c, range(3)), _state(ref, range(3))), (order, n, s)
        c.reset([0, 1, 2])
        assert c.freePages == free
    # in one call: whoever is last keeps the page
    import torch
    for forked, ends, copies, freed in (([256, 256], [210, 166, 166], 2, 1), ([300, 300], [200, 200, 200], 2, 3)):
        c = _cache([T, 0, 0], 8, 2, 64, dtype, bits)
        k, v = _tokens(gpu, c, 1, 1, T)
        c.append(k, v, seq_ids=[0])
        c.fork([0, 0], [1, 2], forked)
        before, free = _state(c, range(3)), c.freePages
        c.trim(90 if forked[0] == 256 else 100, seq_ids=[0, 1, 2])
        assert [c.seqLen(s) for s in range(3)] == ends and c.freePages == free - copies + freed
        assert len({c.seqPages(s)[e // 64] for s, e in enumerate(ends)}) == 3
        for a, b, n in zip(_state(c, range(3)), before, ends):
            assert all(torch.equal(x, y[:, :, :n]) for x, y in zip(a[:-1], b[:-1]))


def test_exhausted_pool(gpu):
    """Forks and trims that would need pages which are not there change
    nothing; a trim may use the pages that it lets go itself."""
    import bsattn
    c = _cache([256] * 4, 8, 2, 64, "f16", num_pages=5)
    k, v = _tokens(gpu, c, 1, 1, 250)
    c.append(k, v, seq_ids=[0])
    c.fork([0], [1], [192])
    assert c.freePages == 1
    with pytest.raises(bsattn.BsattnError) as e:
        c.fork([0, 0], [2, 3], [100, 250])
    assert e.value.code == -3 and c.freePages == 1 and c.seqLen(2) == 0
    c.fork([0], [2])
    assert c.freePages == 0
    state = _state(c, range(4))
    with pytest.raises(bsattn.BsattnError) as e:
        c.trim(100, seq_ids=[1])        # ends inside block 1, which 0 and 2 hold
    assert e.value.code == -3 and _same(state, _state(c, range(4)))
    c.trim(100, seq_ids=[0])            # frees its fourth page, takes it for its copy of block 2
    assert c.seqLen(0) == 150 and c.freePages == 0
    import torch
    assert torch.equal(c.export([0])[0], k[:, :, :150]) and torch.equal(c.export([2])[0], k)
    c.reset([0, 1, 2])
    assert c.freePages == 5


def test_many_and_partial(gpu):
    """More pairs than a launch takes, prefixes of several lengths, several
    sources, and chains of forks."""
    import torch
    n = 70
    c = _cache([500, 129] + [0] * (n + 2), 8, 2, 32, "bf16")
    _fill(gpu, c, [500, 129], 4)
    src = [i % 2 for i in range(n)]
    tokens = [(i * 37) % (500 if i % 2 == 0 else 130) for i in range(n)]
    c.fork(src, list(range(2, n + 2)), tokens)
    c.fork([n], [n + 2], [min(64, c.seqLen(n))])
    full = [c.export([s]) for s in range(2)]
    for i in range(n):
        if tokens[i]:
            k, v = c.export([i + 2])
            assert torch.equal(k, full[i % 2][0][:, :, :tokens[i]]) and torch.equal(v, full[i % 2][1][:, :, :tokens[i]])
            assert torch.equal(c.exportSummaries(i + 2), c.exportSummaries(i % 2)[:, :tokens[i] // 32])
    q = _randn(gpu, 8, (n, 8, 1, D), "bf16")
    ids = list(range(2, n + 2))
    _check(c.decodeDense(q, SCALE, seq_ids=ids), _reference(c, q, ids=ids), "bf16")
    d = c.copy()
    d.reset([0, 1])
    c.reset(ids)
    ids = [s for s in ids if d.seqLen(s)]
    assert all(torch.equal(d.export([s])[0], full[s % 2][0][:, :, :d.seqLen(s)]) for s in ids)
    d.reset(list(range(n + 4)))
    assert d.freePages == d.desc.max_seqs * d.desc.max_blocks_per_seq


@pytest.mark.parametrize("dtype,bits", KINDS)
def test_pages_far_apart(gpu, dtype, bits):
    """Pages all over a pool of more than 4 GiB: what a small pool gives."""
    import torch
    log(f"[far pages] {dtype} bits={bits}")
    near = _cache([3000] * 10, 32, 8, 64, dtype, bits)
    page = 64 * 8 * {0: 512, 4: 144, 8: 272}[bits]
    far = _cache([3000] * 10, 32, 8, 64, dtype, bits, num_pages=(5 << 30) // page)
    far.shuffleFreePages(3)
    outs = []
    for c in (near, far):
        k, v = (_randn(gpu, i, (1, 8, 2500, D), dtype) for i in (1, 2))
        c.append(k, v, seq_ids=[0])
        c.fork([0] * 8, list(range(1, 9)))
        k, v = (_randn(gpu, i, (9, 8, 1, D), dtype) for i in (3, 4))
        c.append(k, v)
        c.trim(40, seq_ids=[3])
        q = _randn(gpu, 5, (9, 32, 1, D), dtype)
        outs.append((c.decodeDense(q, SCALE), c.decodeDense(q, SCALE, window=1000), c.decode(q, SCALE)))
    assert max(p for s in range(9) for p in far.seqPages(s)) * page > 1 << 32
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_calls_at_once(gpu):
    """Two threads, each with its caches and stream: what one after the other
    gives."""
    import threading
    import torch
    jobs = []
    for i in range(4):
        c = _cache([9000] * 4, 32, 8, 64, "bf16")
        _fill(gpu, c, [8191, 0, 0, 0], 60 + i)
        q = _randn(gpu, 80 + i, (4, 32, 1, D), "bf16")
        jobs.append((c, q))
    torch.cuda.synchronize()

    def work(c, q, out):
        for _ in range(5):
            c.fork([0, 0, 0], [1, 2, 3], [8191, 5000, 63])
            out.append(c.decodeDense(q, SCALE))
            c.reset([1, 2, 3])

    want = []
    for c, q in jobs:
        work(c, q, got := [])
        want.append(got[0])
        assert all(torch.equal(g, got[0]) for g in got)
    torch.cuda.synchronize()
    results = [[] for _ in jobs]

    def thread(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            work(*jobs[i], results[i])
        st.synchronize()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(r) == 5 and all(torch.equal(g, w) for g in r) for r, w in zip(results, want))


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 4), (16, 4), (16, 2), (16, 1)])
def test_shared_prefixes(gpu, dtype, bits, Hq, Hkv):
    """Dense decode of sequences that share their beginnings: branches of two
    prompts and of a branch, in any order beside sequences of their own; more
    of them than one workgroup takes; ends at a block's end; sinks."""
    import torch
    log(f"[shared] {dtype} bits={bits} {Hq}/{Hkv}")
    rows = 32
    c = _cache([2100] * rows, Hq, Hkv, 64, dtype, bits)
    _fill(gpu, c, [1999, 1024, 777] + [0] * (rows - 3), 21, salient=True)
    c.fork([0] * 11, list(range(3, 14)))
    c.fork([1] * 5, list(range(14, 19)))
    k, v = _tokens(gpu, c, 60, 1, 90)
    for s in (3, 5, 15, 17):
        c.append(k, v, seq_ids=[s])
    c.fork([5, 5, 5, 0, 0], [19, 20, 21, 22, 23], [2050, 2089, 1985, 1500, 511])
    c.trim(700, seq_ids=[20])
    g = torch.Generator().manual_seed(4)
    sinks = torch.linspace(-2, 4, Hq, device=gpu)
    for ids in (list(range(3, 14)), list(range(rows)), torch.randperm(rows, generator=g).tolist(), [5, 19], [14, 0, 15],
                [20, 21, 22, 23, 2]):
        q = _randn(gpu, 70 + len(ids), (len(ids), Hq, 1, D), dtype)
        _check(c.decodeDense(q, SCALE, seq_ids=ids), _reference(c, q, ids=ids), dtype, f"{ids}")
        _check(c.decodeDense(q, SCALE, sinks=sinks, seq_ids=ids), _reference(c, q, ids=ids, sinks=sinks), dtype,
               f"sinks {ids}")
        _check(c.decodeDense(q, SCALE, window=900, seq_ids=ids), _reference(c, q, ids=ids, window=900), dtype,
               f"window {ids}")
    # captured, the sequences may be others by the time of a replay
    ids = list(range(3, 14))
    q = _randn(gpu, 90, (len(ids), Hq, 1, D), dtype)
    c.decodeDense(q, SCALE, seq_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.decodeDense(q, SCALE, seq_ids=ids)
    for step in range(3):
        graph.replay()
        _check(out, _reference(c, q, ids=ids), dtype, f"replay {step}")
        c.trim(600, seq_ids=[4 + step])
        k, v = _tokens(gpu, c, 80 + step, 1, 500)
        c.append(k, v, seq_ids=[4 + step])


def test_steps_after_forks(gpu):
    """Reserved, captured steps of branches: no branch writes a page that
    another holds."""
    import torch
    c = _cache([70, 0, 0], 8, 2, 32, "f16", spare=40)
    ref = _cache([70, 70, 70], 8, 2, 32, "f16", spare=40)
    k, v = _tokens(gpu, c, 1, 1, 70)
    c.append(k, v, seq_ids=[0])
    c.fork([0, 0], [1, 2])
    for b in range(3):
        ref.append(k, v, seq_ids=[b])
    ks, vs = _tokens(gpu, c, 5, 3)
    q = _randn(gpu, 9, (3, 8, 1, D), "f16")
    graphs = []
    for x in (c, ref):
        x.reserve(30, seq_ids=[0, 1, 2])
        x.decodeDense(q, SCALE)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.appendStep(ks, vs)
            out = x.decodeDense(q, SCALE), x.decode(q, SCALE)
        graphs.append((g, out))
    for step in range(25):
        a, b = _tokens(gpu, c, 30 + 2 * step, 3)
        ks.copy_(a)
        vs.copy_(b)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1][1], graphs[1][1][1]), f"step {step}"
    c.sync()
    ref.sync()
    _check(graphs[0][1][0], _reference(ref, q), "f16")
    assert _same(_state(c, range(3)), _state(ref, range(3)))


@pytest.mark.parametrize("dtype,bits", KINDS)
def test_the_operators_together(gpu, dtype, bits):
    """Four samples of one prompt: the prompt's projections normed, rotated and
    prefilled, branched, then three steps of every sample: norms, positions at
    the branches' own lengths, append, dense attention, windowed attention with
    sinks.  Each result against the steps in 64 bits on what went in."""
    import torch
    import bsattn
    T, n, Hq, Hkv = 333, 4, 16, 4
    log(f"[together] {dtype} bits={bits}")
    c = _cache([T + 3] * (n + 1), Hq, Hkv, 64, dtype, bits)
    rope = bsattn.initializeRope(64, 500000.0, False, {"rope_type": "linear", "factor": 2.0})
    qw, kw = (_randn(gpu, 70 + i, (D,), dtype) for i in range(2))
    norms = (qw, kw, 1e-6, 1.0)

    def split(p):
        p = p.transpose(1, 2)
        return p[:, :Hq], p[:, Hq:Hq + Hkv], p[:, Hq + Hkv:].contiguous()

    q, k, v = split(_randn(gpu, 1, (1, T, Hq + 2 * Hkv, D), dtype))
    # the prompt is row n of the cache; rows 0 .. n - 1 are its samples
    qr, kr = c.normRotate(q, k, qw, kw, 1e-6, rope, seq_ids=[n], weightOffset=1.0)
    c.append(kr, v, seq_ids=[n])
    c.prefill(qr, SCALE, seq_ids=[n])
    c.fork([n] * n, list(range(n)))
    sinks = torch.linspace(-2, 3, Hq, device=gpu)
    for step in range(3):
        q, k, v = split(_randn(gpu, 10 + step, (n, 1, Hq + 2 * Hkv, D), dtype))
        pos = torch.full((n, 1), T + step, dtype=torch.int32, device=gpu)
        want_q, want_k = c.normRotate(q, k, qw, kw, 1e-6, rope, positions=pos, weightOffset=1.0)
        out = bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, dense=True, rope=rope, norms=norms)
        assert [c.seqLen(b) for b in range(n + 1)] == [T + step + 1] * n + [T]
        if not bits:
            assert all(torch.equal(c.export([b])[0][0, :, -1], want_k[b, :, 0]) for b in range(n))
        _check(out, _reference(c, want_q), dtype, f"step {step}")
        win = c.decodeDense(want_q, SCALE, window=100, sinks=sinks)
        _check(win, _reference(c, want_q, window=100, sinks=sinks), dtype, f"step {step} window")
        # the block-sparse step from the same rotated projections
        c.trim(1, seq_ids=list(range(n)))
        sparse = bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, rope=rope, norms=norms)
        assert torch.equal(sparse, c.decode(want_q, SCALE))
    c.reset(list(range(n)))
    # several tokens at once, dense: the prompt kernel
    q, k, v = split(_randn(gpu, 30, (n, 5, Hq + 2 * Hkv, D), dtype))
    out = bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, "causal", dense=True, rope=rope)
    pos = torch.arange(5, dtype=torch.int32, device=gpu).expand(n, 5).contiguous()
    rot = c.normRotate(q, k, None, None, 0.0, rope, positions=pos)[0]
    assert torch.equal(rot, bsattn.applyRotaryPosition(rope, q, c, positions=pos))
    # (the prompt kernel's bar: 2e-3 over 16-bit caches, 1e-2 over quantized ones, beside its rounding)
    want = _reference(c, rot[:, :, 4:].contiguous())
    err = (out[:, :, 4].double() - want).abs() - (2.0 ** -8 if dtype == "bf16" else 2.0 ** -11) * want.abs()
    assert err.max() <= (1e-2 if bits else 2e-3)


def test_refusals(gpu):
    import torch
    import bsattn
    c = _cache([100] * 4, 8, 2, 32, "f16", spare=32)
    _fill(gpu, c, [100, 40], 1)
    before = c.freePages
    cases = [([0], [0], None), ([0], [1], None), ([0, 0], [2, 2], None), ([4], [2], None), ([0], [4], None),
             ([-1], [2], None), ([0], [2], [101]), ([0], [2], [-1]), ([2], [2], None), ([2, 3], [3, 2], None)]
    for src, dst, n in cases:
        with pytest.raises(bsattn.BsattnError):
            c.fork(src, dst, n)
    with pytest.raises(ValueError):
        c.fork([0, 0], [2])
    with pytest.raises(ValueError):
        c.fork([0], [2], [1, 2])
    with pytest.raises(bsattn.BsattnError):
        c.fork([], [])
    c.reserve(3, seq_ids=[3])
    with pytest.raises(bsattn.BsattnError):
        c.fork([0], [3])                      # holds reserved pages
    c.reset([3])
    k, v = _tokens(gpu, c, 1, 1)
    c.reserve(1, seq_ids=[1])
    c.appendStep(k, v, seq_ids=[1])
    with pytest.raises(bsattn.BsattnError):
        c.fork([0], [2])                      # lengths not read back
    c.sync()
    c.fork([0], [2])
    c.reset([2])
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=gpu)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(bsattn.BsattnError):
            c.fork([0], [2])
    assert c.seqLen(2) == 0 and c.freePages == before
    # attention's own checks come before anything is appended
    q = _randn(gpu, 4, (2, 8, 1, D), "f16")
    k, v = _tokens(gpu, c, 1, 2)
    lens = [c.seqLen(s) for s in range(4)]
    rope = bsattn.RoPE(128)
    bad = [dict(window=5), dict(sinks=torch.zeros(8, device=gpu)), dict(dense=True, window=0),
           dict(dense=True, sinks=torch.zeros(4, device=gpu)), dict(norms=(None, None, 0.0))]
    for kw in bad:
        with pytest.raises(ValueError):
            bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, **kw)
    with pytest.raises(ValueError):
        bsattn.attentionWithCacheUpdate(q[:1].contiguous(), k, v, c, SCALE, dense=True)
    with pytest.raises(ValueError):
        c.normRotate(q, k, torch.zeros(D, dtype=torch.float16, device=gpu), None, 1e-6, rope)
    k2, v2 = _tokens(gpu, c, 1, 2, 3)
    with pytest.raises(ValueError):
        bsattn.attentionWithCacheUpdate(_randn(gpu, 4, (2, 8, 3, D), "f16"), k2, v2, c, SCALE, "causal", dense=True,
                                        window=4)
    assert [c.seqLen(s) for s in range(4)] == lens
