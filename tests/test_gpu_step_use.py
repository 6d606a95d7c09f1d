"""Verification steps as a serving program runs them: rounds of drafts over
several layers against decodes token by token, captured rounds replayed with
eager work between, streams and threads, forks, large pools and strides; and
values at the edges of the types."""
from __future__ import annotations

import math
import threading

import pytest

from common import log
from test_gpu_dense import D, HALF_STEP, KINDS, SCALE, _cache, _check, _dt, _fill, _held, _randn
from test_gpu_step import (_ints, _paths, _plain_append, _rows, _same, _state, _step, _tree, _tree_reference,
                           _verify)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# rounds
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("window", [None, 40])
def test_rounds_of_layers(gpu, dtype, bits, window):
    """Four rounds over three layers, with rotary positions of the drafts' depths and views into one projection: each
    accepted path's outputs are those of the formula over caches that were given its tokens alone, in order."""
    import bsattn
    import torch
    log(f"[rounds] {dtype} bits={bits} window={window}")
    lens, Hq, Hkv, layers, N = [5, 64, 0, 130], 8, 2, 3, 12
    caches, refs = ([_cache(lens, Hq, Hkv, 32, dtype, bits, spare=100) for _ in range(layers)] for _ in range(2))
    for x, (c, r) in enumerate(zip(caches, refs)):
        _fill(gpu, c, lens, 30 + x)
        _fill(gpu, r, lens, 30 + x)
        c.reserve(100, seq_ids=range(4))  # (an empty sequence among them)
    rope = bsattn.RoPE(D, base=10000.0, device=0)
    step = bsattn.Step(caches, rows=4 * N, maxTokens=N)
    held = list(lens)
    for turn in range(4):
        counts = [N, (5 * turn) % (N + 1), 1, N - turn]
        trees = [_tree(40 * turn + i, n) for i, n in enumerate(counts)]
        flat = [p for t in trees for p in t]
        step.map(_ints(gpu, counts), _ints(gpu, flat + [-1] * (step.rows - len(flat))))
        kept = [max(_paths(t), key=len)[:1 + turn] if t else [] for t in trees]
        for x, (c, r) in enumerate(zip(caches, refs)):
            q, k, v = _rows(gpu, c, 1000 * turn + x, step.rows)
            qr, kr = c.normRotate(q.transpose(0, 1)[None], k.transpose(0, 1)[None], None, None, 1e-6, rope,
                                  positions=step.positions[None])
            qr, kr = qr[0].transpose(0, 1), kr[0].transpose(0, 1)
            out = bsattn.attentionWithCacheUpdate(qr, kr, v, c, SCALE, step=step, window=window)
            c.keep(step, _ints(gpu, [p + [0] * (N - len(p)) for p in kept]), _ints(gpu, [len(p) for p in kept]))
            # the reference: the path's tokens one by one
            want, at = [], []
            for i, path in enumerate(kept):
                first = sum(counts[:i])
                for j in path:
                    row = first + j
                    pos = _ints(gpu, [[r.seqLen(i)]])
                    q1, k1 = r.normRotate(q[row][None, :, None], k[row][None, :, None], None, None, 1e-6, rope, positions=pos)
                    assert torch.equal(q1[0, :, 0], qr[row]) and torch.equal(k1[0, :, 0], kr[row])
                    r.append(k1, v[row][None, :, None].contiguous(), seq_ids=[i])
                    ks, vs = _held(r, i)
                    since = max(0, r.seqLen(i) - window) if window else 0
                    o = []
                    for h in range(Hkv):
                        s = q1[0, 4 * h:4 * h + 4, 0].double() @ ks[h, since:].t() * SCALE
                        o.append(torch.softmax(s, -1) @ vs[h, since:])
                    want.append(torch.cat(o))
                    at.append(row)
            _check(out[at][:, :, None], torch.stack(want), dtype, f"turn {turn} layer {x}")
            r.sync()
        held = [a + len(p) for a, p in zip(held, kept)]
    for c, r in zip(caches, refs):
        c.sync()
        assert [c.seqLen(b) for b in range(4)] == held
        assert _same(_state(c, range(4)), _state(r, range(4)))


@pytest.mark.parametrize("dtype,bits,N", [("bf16", 0, 16), ("f16", 0, 5), ("f16", 8, 40), ("f16", 4, 64)])
def test_captured_rounds(gpu, dtype, bits, N):
    """A whole round captured once and replayed over changing counts, trees and accepted paths, well past the lengths
    that it was captured at (further reservations in between); eager rounds of a second cache beside it, with the same
    results bit for bit."""
    import bsattn
    import torch
    log(f"[captured] {dtype} bits={bits} N={N}")
    B, Hq, Hkv = 3, 8, 2
    a, b = (_cache([4000] * B, Hq, Hkv, 64, dtype, bits) for _ in range(2))
    for c in (a, b):
        _fill(gpu, c, [100, 1, 700], 3)
        c.reserve(N)
    steps = [bsattn.Step([c], rows=B * N, maxTokens=N) for c in (a, b)]
    counts, parents = _ints(gpu, [N] * B), _ints(gpu, [-1] * (B * N))
    kept, many = _ints(gpu, [list(range(N))] * B), _ints(gpu, [0] * B)
    q, k, v = _rows(gpu, a, 1, B * N, fused=False)

    def round_(c, step, out):
        step.map(counts, parents)
        c.appendPacked(k, v, step)
        c.attendTree(q, step, SCALE, out=out)
        c.keep(step, kept, many)

    outs = [torch.zeros(B * N, Hq, D, dtype=_dt(dtype), device=gpu) for _ in range(2)]
    round_(a, steps[0], outs[0])  # (many: none is kept)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        round_(a, steps[0], outs[0])
    for turn in range(12):
        n = [(7 * turn + 3 * i) % (N + 1) for i in range(B)]
        trees = [_tree(100 * turn + i, x, 0.1) for i, x in enumerate(n)]
        flat = [p for t in trees for p in t]
        paths = [max(_paths(t), key=len) if t else [] for t in trees]
        counts.copy_(_ints(gpu, n))
        parents.copy_(_ints(gpu, flat + [0] * (B * N - len(flat))))
        kept.copy_(_ints(gpu, [p + [0] * (N - len(p)) for p in paths]))
        many.copy_(_ints(gpu, [len(p) for p in paths]))
        for x, y in zip((q, k, v), _rows(gpu, a, 50 + turn, B * N, fused=False)):
            x.copy_(y)
        for o in outs:
            o.fill_(5)
        g.replay()
        round_(b, steps[1], outs[1])
        torch.cuda.synchronize()
        for x in ("starts", "taken", "requests", "positions", "ancestors", "ends"):
            assert torch.equal(getattr(steps[0], x), getattr(steps[1], x)), (turn, x)
        held = steps[0].taken.sum().item()
        assert held == sum(n)
        # (the parts of the replayed launch are those of the lengths at its capture: another order of sums, and so
        # two roundings, each within _check's bound)
        one, two = outs[0][:held].double(), outs[1][:held].double()
        h, rms = HALF_STEP[dtype], two.pow(2).mean(-1, keepdim=True).sqrt()
        assert ((one - two).abs() <= 2 * (h * torch.maximum(one.abs(), two.abs()) + 1.8 * h * rms + 2.0 ** -25)).all(), turn
        assert (outs[0][held:] == 5).all() and (outs[1][held:] == 5).all()
        # the host's turn: lengths, another reservation, now and then a long prompt between
        for c in (a, b):
            c.sync()
            if turn == 5:
                c.append(*(_randn(gpu, 77 + x, (B, Hkv, 2500, D), "f16" if bits else dtype) for x in (0, 1)))
            c.reserve(N)
        assert [a.seqLen(i) for i in range(B)] == [b.seqLen(i) for i in range(B)]
        assert _same(_state(a, range(B)), _state(b, range(B)))


@pytest.mark.parametrize("what", ["append", "map"])
def test_captured_parts_of_rounds(gpu, what):
    """The append and attention captured, with or without the map, and the rest of each round eager, host calls between
    the rounds: states of a cache that was given the kept tokens."""
    import bsattn
    import torch
    log(f"[captured parts] {what}")
    B, N = 2, 9
    c, ref = (_cache([600] * B, 8, 2, 32, "bf16") for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, [50, 333], 3)
    c.reserve(64)
    step = bsattn.Step([c], rows=B * N, maxTokens=N)
    counts, kept, many = _ints(gpu, [N, N]), _ints(gpu, [[0, 2, 5]] * B), _ints(gpu, [0, 0])
    q, k, v = _rows(gpu, c, 1, B * N, fused=False)
    out = torch.zeros_like(q)

    def first():
        c.appendPacked(k, v, step)
        c.attendTree(q, step, SCALE, out=out)

    step.map(counts)
    first()
    c.keep(step, kept, many)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    if what == "append":
        step.map(counts)
    with torch.cuda.graph(g):
        if what == "map":
            step.map(counts)
        first()
    for turn in range(6):
        n = [(3 * turn + i) % (N + 1) for i in range(B)]
        counts.copy_(_ints(gpu, n))
        many.copy_(_ints(gpu, [min(3, x // 2) for x in n]))
        for x, y in zip((q, k, v), _rows(gpu, c, 20 + turn, B * N, fused=False)):
            x.copy_(y)
        c.sync()
        if turn in (2, 4):  # (the host's calls between the rounds)
            more = [_randn(gpu, 70 + turn + x, (B, 2, 3, D), "bf16") for x in (0, 1)]
            for x in (c, ref):
                x.append(*more)
                x.trim(1)
            c.reserve(64)
        lens = [c.seqLen(b) for b in range(B)]
        if what == "append":
            step.map(counts)
        out.fill_(7)
        g.replay()
        c.sync()
        assert [c.seqLen(b) for b in range(B)] == [x + y for x, y in zip(lens, n)]
        held = sum(n)
        if held:
            _check(out[:held, :, None], _tree_reference(c, q, step, lens, n, None)[:held], "bf16", f"turn {turn}")
        assert (out[held:] == 7).all()
        c.keep(step, kept, many)
        c.sync()
        for b in range(B):
            path = [0, 2, 5][:min(3, n[b] // 2)]
            at = torch.tensor([sum(n[:b]) + x for x in path], dtype=torch.long, device=gpu)
            _plain_append(ref, k[at], v[at], b)
            assert c.seqLen(b) == lens[b] + len(path)
        assert _same(_state(c, range(B)), _state(ref, range(B))), turn


def test_two_graphs_of_a_cache(gpu):
    """Two captured attentions of one cache, replayed in turn on a stream, share its workspace: each replay is right."""
    import torch
    log("[two graphs]")
    c = _cache([9000, 3000], 16, 2, 64, "bf16", spare=64)
    _fill(gpu, c, [9000, 3000], 3)
    step = _step(gpu, [c], [40, 64], None)
    q, k, v = _rows(gpu, c, 5, step.rows, fused=False)
    c.appendPacked(k, v, step)
    base = [c.attendTree(q, step, SCALE), c.attendTree(-q, step, SCALE, window=500)]
    torch.cuda.synchronize()
    graphs = []
    for x, w in ((q, None), ((-q).contiguous(), 500)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.attendTree(x, step, SCALE, window=w)
        graphs.append((g, out, x))
    for _ in range(4):
        for (g, out, _), want in zip(graphs, base):
            out.fill_(3)
            g.replay()
            eager = c.attendTree(q, step, SCALE)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(eager, base[0])


def test_streams_and_threads(gpu):
    """Four caches attended to from four threads on streams of their own, many times over, with split sequences: the
    results are those of one at a time."""
    import torch
    log("[streams]")
    work = []
    for x, (dtype, bits) in enumerate(KINDS):
        c = _cache([6000, 50], 8, 2, 64, dtype, bits, spare=64)
        _fill(gpu, c, [6000, 50], 3 + x)
        step = _step(gpu, [c], [30, 64], [_tree(x, 30), _tree(9 + x, 64)])
        q, k, v = _rows(gpu, c, 5 + x, step.rows, fused=False)
        c.appendPacked(k, v, step)
        work.append((c, step, q, c.attendTree(q, step, SCALE)))
    torch.cuda.synchronize()
    wrong = []

    def run(c, step, q, want):
        with torch.cuda.device(0), torch.cuda.stream(torch.cuda.Stream()):
            outs = [c.attendTree(q, step, SCALE) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(o, want) for o in outs):
                wrong.append(c)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_threads_map_steps(gpu):
    """Maps from several threads: every step names its own cache's state."""
    import torch
    log("[threads map]")
    caches = [_cache([40], 2, 1, 32, "f16", spare=300) for _ in range(4)]
    for x, c in enumerate(caches):
        _fill(gpu, c, [40], x)
        c.reserve(300)
    torch.cuda.synchronize()
    wrong = []

    def run(c, seed):
        import bsattn
        with torch.cuda.device(0), torch.cuda.stream(torch.cuda.Stream()):
            step, held = bsattn.Step([c], rows=8, maxTokens=8), 40
            kept = _ints(gpu, [list(range(8))])
            for turn in range(30):
                n = 1 + (seed + turn) % 8
                step.map(_ints(gpu, [n]))
                _, k, v = _rows(gpu, c, turn, 8, fused=False)
                c.appendPacked(k, v, step)
                c.keep(step, kept, _ints(gpu, [n - n // 2]))
                held += n - n // 2
            c.sync()
            if c.seqLen(0) != held:
                wrong.append((seed, held, c.seqLen(0)))

    threads = [threading.Thread(target=run, args=(c, i)) for i, c in enumerate(caches)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---------------------------------------------------------------------------
# forks, large pools, strides
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", KINDS)
def test_forks_take_steps(gpu, dtype, bits):
    """Branches of a prompt take trees and keep paths by themselves; the prompt's pages stay as they were."""
    import torch
    log(f"[forks] {dtype} bits={bits}")
    lens = [150, 0, 0, 0]
    c, ref = (_cache([150] * 4, 8, 2, 64, dtype, bits, spare=64) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, lens, 3)
        x.fork([0, 0, 0], [1, 2, 3])
    c.trim(30, seq_ids=[2])  # (ends inside a shared block)
    ref.trim(30, seq_ids=[2])
    before = _state(c, [0])
    counts = [0, 20, 33, 7]
    trees = [_tree(i, n) for i, n in enumerate(counts)]
    step = _verify(gpu, c, [150, 150, 120, 150], counts, trees, 11)
    _, k, v = _rows(gpu, c, 11, step.rows)
    kept = [[], [0, 1], max(_paths(trees[2]), key=len), [0]]
    c.keep(step, _ints(gpu, [p + [0] * (64 - len(p)) for p in kept]), _ints(gpu, [len(p) for p in kept]))
    c.sync()
    for i, p in enumerate(kept):
        at = torch.tensor([sum(counts[:i]) + j for j in p], dtype=torch.long, device=gpu)
        _plain_append(ref, k[at], v[at], i)
    assert _same(_state(c, [0]), before)
    assert _same(_state(c, range(4)), _state(ref, range(4)))


@pytest.mark.parametrize("dtype,bits", [("bf16", 0), ("f16", 8)])
def test_large_pool(gpu, dtype, bits):
    """Pages more than 2^32 bytes (and elements of 16 bits) into the pool."""
    import bsattn
    log(f"[large pool] {dtype} bits={bits}")
    Hq, Hkv, Tb = 16, 8, 64
    slab = 2 * Tb * D * (2 if not bits else 1)
    pages = (10 << 30) // (Hkv * slab)
    fill = -(-pages // 12288)  # sequences that hold the rest of it
    c = bsattn.BlockSparseKVCache(max_seqs=2 + fill, num_q_heads=Hq, num_kv_heads=Hkv, block_size=Tb, dtype=_dt(dtype), kv_bits=bits,
                                  top_k=2, max_blocks_per_seq=12288, num_pages=pages, device=0)
    c.shuffleFreePages(3)
    for b in range(fill):
        c.reserve(min(12288, c.freePages - 40) * Tb, seq_ids=[b])
    assert c.freePages == 40
    lens, counts, ids = [700, 90], [33, 20], [fill, fill + 1]
    for b, n in zip(ids, lens):
        c.append(*(_randn(gpu, 5 + b + x, (1, Hkv, n, D), "f16" if bits else dtype) for x in (0, 1)), seq_ids=[b])
    assert max(p for b in ids for p in c.seqPages(b)) * Hkv * slab > 1 << 33
    trees = [_tree(i, n) for i, n in enumerate(counts)]
    step = _verify(gpu, c, lens, counts, trees, 7, ids=ids)
    paths = [max(_paths(t), key=len) for t in trees]
    kept = [list(c.seqPages(b)) for b in ids]
    c.keep(step, _ints(gpu, [p + [0] * (33 - len(p)) for p in paths]), _ints(gpu, [len(p) for p in paths]))
    c.sync()
    assert [c.seqLen(b) for b in ids] == [n + len(p) for n, p in zip(lens, paths)]
    assert [list(c.seqPages(b)) for b in ids] == kept


def test_far_rows(gpu):
    """Rows of queries, keys and values more than 2^31 elements apart from the first."""
    import torch
    log("[far rows]")
    N, far = 20, 1 << 27
    c, ref = (_cache([50], 4, 2, 32, "bf16", spare=32) for _ in range(2))
    for x in (c, ref):
        _fill(gpu, x, [50], 5)
    flat = torch.empty(N * far, dtype=torch.bfloat16, device=gpu)
    wide = flat.view(N, far)[:, :8 * D].view(N, 8, D)
    assert wide.stride(0) * (N - 1) > 1 << 31
    wide.copy_(_randn(gpu, 3, (N, 8, D), "bf16"))
    out = []
    for x, rows in ((c, wide), (ref, wide.contiguous())):
        step = _step(gpu, [x], [N], [_tree(3, N)])
        x.appendPacked(rows[:, 4:6], rows[:, 6:8], step)
        out.append(x.attendTree(rows[:, :4], step, SCALE))
        x.sync()
    assert torch.equal(*out) and _same(_state(c, [0]), _state(ref, [0]))


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv,counts", [(16, 1, [64, 20, 33]), (32, 2, [17, 64, 1]), (8, 1, [12, 24, 9]),
                                           (4, 1, [10, 11, 25]), (32, 16, [33, 9, 41])])
def test_column_groups(gpu, dtype, bits, Hq, Hkv, counts):
    """Columns of one to four groups of workgroups, and numbers of column tiles that waves hold one, two or none of."""
    log(f"[groups] {dtype} bits={bits} {Hq}/{Hkv} {counts}")
    lens = [3000, 45, 64]
    c = _cache(lens, Hq, Hkv, 64, dtype, bits, spare=64)
    _fill(gpu, c, lens, 5)
    _verify(gpu, c, lens, counts, [_tree(i, n) for i, n in enumerate(counts)], 9)


# ---------------------------------------------------------------------------
# values
# ---------------------------------------------------------------------------
def _values(gpu, kind, shape, seed):
    """Values in bf16 of a kind, [..., tokens, D]."""
    import torch
    v = _randn(gpu, seed, shape, "f16").float()
    T = shape[-2]
    if kind == "dims":  # (dims of very different sizes)
        v *= 10.0 ** (torch.arange(D, device=gpu) % 9 - 6)
    elif kind == "tiny":
        v *= 2.0 ** -30
    elif kind == "huge":
        v *= 2.0 ** 90
    elif kind == "some huge":  # (past fp16's range in a few tokens)
        v[..., 5::97, :] *= 1e6
    elif kind == "zeros":
        v[..., 40:200, :] = 0
        v[..., ::3] = 0
    elif kind == "tokens":  # (tokens of very different sizes)
        v *= 2.0 ** -(8.0 * (torch.arange(T, device=gpu) % 4))[:, None]
    elif kind == "steps":  # (about the sizes where another form is taken)
        v = torch.sign(v) * 2.0 ** (torch.arange(D, device=gpu) % 30 - 14)
    return v.to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["dims", "tiny", "huge", "some huge", "zeros", "tokens", "steps"])
@pytest.mark.parametrize("N", [4, 8, 16, 40])
def test_value_ranges(gpu, kind, N):
    """bf16 values that fp16 does not hold, or holds in part: columns of every width (16 heads of 2)."""
    log(f"[values] {kind} N={N}")
    _check_values(gpu, kind, N, 700, 16, 2)


@pytest.mark.parametrize("kind", ["dims", "some huge", "zeros", "tokens"])
@pytest.mark.parametrize("N", [16, 32])
def test_value_ranges_of_long_sequences(gpu, kind, N):
    """The same where workgroups have many units (64 and 128 columns in waves of two column tiles)."""
    log(f"[values, long] {kind} N={N}")
    _check_values(gpu, kind, N, 20000, 32, 8)


def _check_values(gpu, kind, N, T, Hq, Hkv):
    import torch
    G = Hq // Hkv
    c = _cache([T], Hq, Hkv, 64, "bf16", spare=64)
    c.append(_randn(gpu, 3, (1, Hkv, T, D), "bf16"), _values(gpu, kind, (1, Hkv, T, D), 4))
    step = _step(gpu, [c], [N], [_tree(3, N)])
    q, k, _ = _rows(gpu, c, 8, N, fused=False)
    v = _values(gpu, kind, (Hkv, N, D), 6).transpose(0, 1).contiguous()
    c.appendPacked(k, v, step)
    out = c.attendTree(q, step, SCALE).double()
    c.sync()
    want = _tree_reference(c, q, step, [T], [N], [_tree(3, N)])
    keys, vals = _held(c, 0)
    # weights are rounded to fp16's 11 bits, half a step 2^-12, and their sum with them; scores and sums in 32
    # bits add less than that again: 2^-11 of the weights' sum of magnitudes in all.  Where a dim has a value of
    # 2^-10 or more, those below 2^-14 beside it may be multiples of 2^-24: 2^-25 each, for weights that add to 1
    reach = torch.zeros_like(want)
    paths = _paths(_tree(3, N))
    for h in range(Hkv):
        for j, path in enumerate(paths):
            on = list(range(T)) + [T + a for a in path]
            p = torch.softmax(q[j, G * h:G * h + G].double() @ keys[h][on].t() * SCALE, -1)
            reach[j, G * h:G * h + G] = p @ vals[h][on].abs()
    top = vals.abs().amax(1).repeat_interleave(G, 0)[None]  # [1, Hq, D]
    tol = HALF_STEP["bf16"] * want.abs() + 2.0 ** -11 * reach + torch.where(top >= 2.0 ** -10, 2.0 ** -25, 0.0)
    worst = ((out - want).abs() / tol.clamp_min(1e-300)).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("scale", [2.0 ** -14, 2.0 ** 8, 200.0])
def test_affine_scales(gpu, bits, scale):
    """Values whose scales are near the ends of fp16: the output's error is that of its rounding."""
    import torch
    log(f"[affine] bits={bits} {scale}")
    T, N, Hkv = 500, 24, 2
    c = _cache([T], 8, Hkv, 64, "f16", bits, spare=64)
    size = scale * (1 if bits == 4 else 16)
    c.append(_randn(gpu, 3, (1, Hkv, T, D), "f16"), (_randn(gpu, 4, (1, Hkv, T, D), "f16").float() * size).half())
    step = _step(gpu, [c], [N], [_tree(3, N)])
    q, k, v = _rows(gpu, c, 8, N, fused=False)
    c.appendPacked(k, (v.float() * size).half(), step)
    out = c.attendTree(q, step, SCALE)
    c.sync()
    _check(out[:, :, None], _tree_reference(c, q, step, [T], [N], [_tree(3, N)]), "f16", f"{bits} {scale}")


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales(gpu, dtype, bits, scale):
    """Negative scales, none (the mean of what is seen) and large ones (one token has all the weight)."""
    import torch
    log(f"[scales] {dtype} bits={bits} {scale}")
    lens, counts = [300, 2000], [9, 30]
    trees = [_tree(i, n) for i, n in enumerate(counts)]
    c = _cache(lens, 8, 2, 64, dtype, bits, spare=64)
    _fill(gpu, c, lens, 5)
    step = _step(gpu, [c], counts, trees)
    q, k, v = _rows(gpu, c, 8, step.rows, fused=False)
    c.appendPacked(k, v, step)
    out = c.attendTree(q, step, scale)
    c.sync()
    want = _tree_reference(c, q, step, lens, counts, trees, scale=scale)
    if scale == 3.0:
        # sums of 128 products in 32 bits are off by 2^-24 of their magnitudes' sum at a step: 128 * 2 / pi for keys
        # of 1, and for codes, as 1024 + c, 128 * 0.8 * 1279 (int8) or 1039 (int4) times their scales of 1 / 40 and 0.45;
        # a weight is off by twice that times the scale, an output by twice that times its largest value, 5
        size = {0: 130, 8: 102 * 1279 / 40, 4: 102 * 1039 * 0.45}[bits]
        err, h = (out.double() - want).abs(), HALF_STEP[dtype]
        rms = want.pow(2).mean(-1, keepdim=True).sqrt()
        assert (err <= h * want.abs() + 1.8 * h * rms + 2 * 5 * 2 * 3.0 * 2.0 ** -24 * size + 2.0 ** -25).all()
    else:
        _check(out[:, :, None], want, dtype, str(scale))


# ---------------------------------------------------------------------------
# refusals and timing
# ---------------------------------------------------------------------------
def test_refusals(gpu):
    """What the Python layer and the library refuse, with nothing changed."""
    import bsattn
    import torch
    log("[refusals]")
    c = _cache([40, 40], 4, 2, 32, "f16", spare=64)
    _fill(gpu, c, [40, 40], 3)
    c.reserve(16)
    step = bsattn.Step([c], rows=16, maxTokens=8)
    q, k, v = _rows(gpu, c, 3, 16, fused=False)
    n2 = _ints(gpu, [3, 4])
    for caches, rows, most in (([], 8, 8), ([c] * 129, 8, 8), ([c], 0, 8), ([c], 8, 0)):
        with pytest.raises(ValueError):
            bsattn.Step(caches, rows=rows, maxTokens=most)
    with pytest.raises(bsattn.BsattnError, match="twice"):
        bsattn.Step([c, c], rows=8, maxTokens=8).map(n2)
    for counts, parents in ((n2.long(), None), (n2.cpu(), None), (n2[None], None), (_ints(gpu, [1, 1, 1]), None),
                            (_ints(gpu, []), None), (n2, _ints(gpu, [0] * 15)), (n2, torch.zeros(16, device=gpu))):
        with pytest.raises(ValueError):
            step.map(counts, parents)
    with pytest.raises(bsattn.BsattnError, match="bsattn_step_map"):
        c.appendPacked(k, v, step)
    step.map(n2)
    with pytest.raises(bsattn.BsattnError, match="bsattn_append_packed"):
        c.attendTree(q, step, SCALE)
    for bad in (k[:15], k.float(), k.cpu(), k[:, :1], k.transpose(1, 2), k.repeat(1, 1, 2)[:, :, ::2],
                torch.empty(16 * 256 + 1, dtype=k.dtype, device=gpu)[1:].view(16, 2, D)):
        with pytest.raises(ValueError):
            c.appendPacked(bad, v, step)
        with pytest.raises(ValueError):
            c.appendPacked(k, bad, step)
    c.appendPacked(k, v, step)
    base = c.attendTree(q, step, SCALE)
    for kw in ({"window": -1}, {"window": 0}, {"sinks": torch.zeros(3, device=gpu)}, {"out": torch.empty_like(q[:8])},
               {"out": torch.empty_like(q).float()}):
        with pytest.raises(ValueError):
            c.attendTree(q, step, SCALE, **kw)
    with pytest.raises(ValueError):
        bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, mask="causal", step=step)
    kept = _ints(gpu, [[0], [0]])
    for a, b in ((kept.long(), n2), (kept[0], n2), (kept, n2[:1]), (kept[:, :0], n2), (kept.cpu(), n2)):
        with pytest.raises(ValueError):
            c.keep(step, a, b)
    assert torch.equal(c.attendTree(q, step, SCALE)[:7], base[:7])  # (the others are nobody's)
    with pytest.raises(bsattn.BsattnError, match="bsattn_sync"):
        c.append(k[:2, :, None].contiguous(), v[:2, :, None].contiguous())
    c.keep(step, kept, _ints(gpu, [1, 1]))
    with pytest.raises(bsattn.BsattnError, match="moved"):
        c.attendTree(q, step, SCALE)
    c.sync()
    assert [c.seqLen(0), c.seqLen(1)] == [41, 41]
    c.trim(1)
    with pytest.raises(bsattn.BsattnError, match="changed"):
        c.appendPacked(k, v, step)
    chunk = bsattn.Step([c], rows=16, maxTokens=65).map(n2)
    with pytest.raises(ValueError):
        bsattn.attentionWithCacheUpdate(q, k, v, c, SCALE, step=chunk)
    with pytest.raises(bsattn.BsattnError, match="64"):
        bsattn.Step([c], rows=16, maxTokens=65).map(n2, _ints(gpu, [-1] * 16))
    c.close()
    with pytest.raises(ValueError):
        step.map(n2)


def test_kernel_times(gpu):
    """Maps, attentions and kept paths are timed under kinds of their own."""
    from bsattn import _lib
    log("[times]")
    c = _cache([4000], 8, 2, 64, "f16", spare=64)
    _fill(gpu, c, [4000], 3)
    c.profile()
    step = _step(gpu, [c], [30], None)
    q, k, v = _rows(gpu, c, 3, 30)
    c.appendPacked(k, v, step)
    c.attendTree(q, step, SCALE)
    c.keep(step, _ints(gpu, [[0]]), _ints(gpu, [1]))
    for kind in (_lib.KERNEL_MAP, _lib.KERNEL_TREE, _lib.KERNEL_KEEP, _lib.KERNEL_APPEND):
        ms, n = c.profileRead(kind)
        assert n == 1 and 0 < ms < 50


# ---------------------------------------------------------------------------
# random shapes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(40))
def test_random_rounds(gpu, seed):
    """Two rounds of seeded random caches, layouts, lengths, counts, trees, windows, sinks, sequence orders and kept
    paths: attention against the formula, states against caches that were given the kept tokens."""
    import random
    import torch
    r = random.Random(seed)
    dtype, bits = r.choice(KINDS)
    Tb, (Hq, Hkv) = r.choice([32, 64]), r.choice([(8, 8), (4, 1), (32, 8), (16, 1), (8, 2), (16, 2), (64, 4), (2, 2)])
    B, most = r.randint(1, 9), r.choice([1, 4, 9, 16, 33, 64])
    lens = [r.choice([0, 1, 31, 32, 63, 64, r.randint(2, 300), r.randint(300, 6000)]) for _ in range(B)]
    log(f"[random {seed}] {dtype} bits={bits} Tb={Tb} {Hq}/{Hkv} most={most} {lens}")
    c, ref = (_cache(lens, Hq, Hkv, Tb, dtype, bits, spare=2 * 64) for _ in range(2))
    salient = r.random() < 0.5
    for x in (c, ref):
        _fill(gpu, x, lens, 1000 + seed, salient=salient)
    for turn in range(2):
        ids = r.sample(range(B), r.randint(1, B))
        counts = [r.choice([0, 1, r.randint(1, most), most]) for _ in ids]
        trees = None if r.random() < 0.25 else [_tree(10 * seed + i, n, r.choice([0, 0.1])) for i, n in enumerate(counts)]
        window = r.choice([None, None, 1, 50, 700])
        sinks = _randn(gpu, seed, (Hq,), "f16").float() if r.random() < 0.4 else None
        step = _verify(gpu, c, [lens[b] for b in ids], counts, trees, 50 * seed + turn, f"{seed} {turn}", ids=ids,
                       window=window, sinks=sinks, rows=max(1, sum(counts)) + r.randint(0, 3), fused=r.random() < 0.5)
        _, k, v = _rows(gpu, c, 50 * seed + turn, step.rows)
        kept = [sorted(r.sample(range(n), r.randint(0, min(n, 12)))) for n in counts]
        width = max(1, max(len(p) for p in kept))
        c.keep(step, _ints(gpu, [p + [0] * (width - len(p)) for p in kept]), _ints(gpu, [len(p) for p in kept]))
        c.sync()
        for i, (b, p) in enumerate(zip(ids, kept)):
            at = torch.tensor([sum(counts[:i]) + j for j in p], dtype=torch.long, device=gpu)
            _plain_append(ref, k[at], v[at], b)
            lens[b] += len(p)
        assert [c.seqLen(b) for b in range(B)] == lens
        assert _same(_state(c, range(B)), _state(ref, range(B))), turn
