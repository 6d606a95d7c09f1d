"""Dense decode (bsattn_decode_dense): one new token per sequence over every
token of its cache or the last `window` ones, with sink logits or without,
against the formula in 64 bits over what the cache holds."""
from __future__ import annotations

import math

import pytest

from common import log

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # eps / 2


def _dt(name):
    import torch
    return torch.float16 if name == "f16" else torch.bfloat16


def _randn(gpu, seed, shape, dtype):
    import torch
    return torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(_dt(dtype))


def _cache(lens, Hq, Hkv, Tb, dtype, bits=0, spare=0, **kw):
    import bsattn
    blocks = max(1, max(-(-(n + spare) // Tb) for n in lens))
    return bsattn.BlockSparseKVCache(max_seqs=len(lens), num_q_heads=Hq, num_kv_heads=Hkv, block_size=Tb,
                                     dtype=_dt(dtype), kv_bits=bits, top_k=2, max_blocks_per_seq=blocks, device=0, **kw)


def _fill(gpu, c, lens, seed, salient=False):
    """Random tokens; returns nothing: the cache's own state is what counts."""
    import torch
    c.shuffleFreePages(seed)
    for b, n in enumerate(lens):
        if not n:
            continue
        k, v = (_randn(gpu, seed + 10 * b + i, (1, c._hkv, n, D), "f16" if c.bits else
                       {torch.float16: "f16", torch.bfloat16: "bf16"}[c.dtype]) for i in (0, 1))
        if salient:
            k[:, :, ::97] *= 4
        c.append(k, v, seq_ids=[b])


def _held(c, b):
    """Keys and values [Hkv, T, D] of sequence b in 64 bits."""
    import torch
    if not c.bits:
        return [x[0].double() for x in c.export([b])]
    out = []
    for w, s, z in c.exportQuantized([b]):
        sh = c.bits * torch.arange(32 // c.bits, device=w.device, dtype=torch.int32)
        code = ((w[0][..., None] >> sh) & ((1 << c.bits) - 1)).double().reshape(*w.shape[1:3], D)
        out.append(code * s[0].double().repeat_interleave(64, -1) + z[0].double().repeat_interleave(64, -1))
    return out


def _reference(c, q, ids=None, window=None, sinks=None, scale=SCALE):
    """[B, Hq, D] in 64 bits."""
    import torch
    B, Hq = q.shape[:2]
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=q.device)
    for i, b in enumerate(ids if ids is not None else range(B)):
        T = c.seqLen(b)
        if T == 0:
            continue
        k, v = _held(c, b)
        if window:
            k, v = k[:, max(0, T - window):], v[:, max(0, T - window):]
        s = torch.matmul(q[i, :, 0].double().reshape(c._hkv, -1, D), k.transpose(1, 2).contiguous()) * scale
        top = s.amax(-1, keepdim=True)
        if sinks is not None:
            sk = sinks.double().reshape(c._hkv, -1, 1)
            top = torch.maximum(top, sk)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sk - top)
        out[i] = (torch.matmul(p, v) / total).reshape(Hq, D)
    return out


def _check(got, want, dtype, what=""):
    """Outputs are rounded once: at most half a step of the value, 0.58 of one
    (a uniform error's share, 1 / sqrt 3) in the mean square.  The rest of the
    arithmetic is held to 0.3 of half a step of the row's root mean square: P
    enters with 2^-18 (bf16) or 2^-22, the scores and sums are fp32 (scores of
    a few units: 2^-19 each), and int4's offset of 1024 against codes of 4.6
    standard deviations costs 2^-24 * 1024 / 4.6 a token, 2^-16: 0.06 of
    fp16's half step at the most.  Six deviations bound the largest.

    fp16 values below 2^-14 are rounded to multiples of 2^-24 instead: an
    error of up to 2^-25 whatever the value, 2^-25 / sqrt 3 in the mean square.
    (Outputs of 4e-5, as codes with scales of 2^-12 give, have a relative
    error of 2^-25 / sqrt 3 / 4e-5 = 4.3e-4 from that alone, 0.88 of 2^-11.)"""
    import torch
    got = got[:, :, 0].double()
    h = HALF_STEP[dtype]
    err = (got - want).abs()
    rms = want.pow(2).mean(-1, keepdim=True).sqrt()
    tol = h * want.abs() + 6 * 0.3 * h * rms + 2.0 ** -25
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance, error {err.max().item():.3g}"
    mean, size = err.pow(2).mean().sqrt().item(), want.pow(2).mean().sqrt().item()
    assert mean <= 0.66 * h * size + 0.58 * 2.0 ** -25, f"{what}: {mean / (h * size):.3g} of half a step in the mean square"
    assert torch.isfinite(got).all()


KINDS = [("f16", 0), ("bf16", 0), ("f16", 4), ("f16", 8)]


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (4, 2), (32, 8), (16, 2), (64, 4), (16, 16), (16, 1)])
@pytest.mark.parametrize("Tb", [32, 64])
def test_lengths(gpu, dtype, bits, Hq, Hkv, Tb):
    """Lengths from nothing to many parts, ends inside units and pages."""
    lens = [1, 0, 2, 31, 32, 33, 63, 64, 65, 127, 129, 500, 1000, 2049, 4500, 5]
    log(f"[dense] {dtype} bits={bits} {Hq}/{Hkv} Tb={Tb}")
    c = _cache(lens, Hq, Hkv, Tb, dtype, bits)
    _fill(gpu, c, lens, 100 + Hq + Tb, salient=True)
    q = _randn(gpu, 7, (len(lens), Hq, 1, D), dtype)
    got = c.decodeDense(q, SCALE)
    assert (got[1] == 0).all()
    _check(got, _reference(c, q), dtype)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("window", [1, 2, 31, 33, 64, 100, 1000, 100000])
def test_window_and_sinks(gpu, dtype, bits, window):
    import torch
    lens = [1, 0, 40, 64, 100, 1001, 3333]
    log(f"[dense] {dtype} bits={bits} window={window}")
    c = _cache(lens, 32, 8, 64, dtype, bits)
    _fill(gpu, c, lens, window)
    q = _randn(gpu, 8, (len(lens), 32, 1, D), dtype)
    sinks = torch.randn(32, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu) * 3
    sinks[5], sinks[6], sinks[7] = -math.inf, 300.0, -300.0
    for sk in (None, sinks):
        got = c.decodeDense(q, SCALE, window=window, sinks=sk)
        assert (got[1] == 0).all()
        _check(got, _reference(c, q, window=window, sinks=sk), dtype, f"sinks {sk is not None}")
    _check(c.decodeDense(q, SCALE, sinks=sinks), _reference(c, q, sinks=sinks), dtype, "no window")


@pytest.mark.parametrize("dtype,bits,B,T,Hq,Hkv,Tb", [
    ("bf16", 0, 2, 32768, 32, 8, 64), ("f16", 0, 1, 100003, 8, 2, 32), ("f16", 4, 1, 131072, 32, 8, 64),
    ("f16", 8, 2, 70001, 64, 4, 32), ("f16", 4, 3, 20000, 64, 4, 64)])
def test_long(gpu, dtype, bits, B, T, Hq, Hkv, Tb):
    log(f"[dense long] {dtype} bits={bits} {B}x{T} {Hq}/{Hkv} Tb={Tb}")
    lens = [T - 777 * b for b in range(B)]
    c = _cache(lens, Hq, Hkv, Tb, dtype, bits)
    _fill(gpu, c, lens, T)
    q = _randn(gpu, 9, (B, Hq, 1, D), dtype)
    _check(c.decodeDense(q, SCALE), _reference(c, q), dtype)


@pytest.mark.parametrize("dtype,bits", KINDS)
def test_what_is_not_seen(gpu, dtype, bits):
    """Pages that held infinities and NaN before, behind the last token; and
    tokens in front of the window that hold them now."""
    import torch
    lens = [70, 37, 1, 200, 5]
    c = _cache([256] * 5, 8, 2, 64, dtype, bits)
    bad = torch.full((5, 2, 256, D), math.inf, dtype=_dt(dtype), device=gpu)
    bad[..., ::3] = math.nan
    if bits:
        kw, ks = c.quantizedShapes(5, 256)
        w = torch.full(kw, -1, dtype=torch.int32, device=gpu)
        s = torch.full(ks, math.nan, dtype=torch.float16, device=gpu)
        c.appendQuantized((w, s, s), (w, s, s))
    else:
        c.append(bad, bad)
    c.reset(list(range(5)))
    _fill(gpu, c, lens, 41)
    q = _randn(gpu, 10, (5, 8, 1, D), dtype)
    _check(c.decodeDense(q, SCALE), _reference(c, q), dtype)
    # a token with a NaN key and infinite values at position 100 of sequence 3
    c.trim(100, seq_ids=[3])
    want = _randn(gpu, 43, (1, 2, 99, D), dtype), _randn(gpu, 44, (1, 2, 99, D), dtype)
    if bits:
        kw, ks = c.quantizedShapes(1, 1)
        w, s = torch.full(kw, -1, dtype=torch.int32, device=gpu), torch.full(ks, math.inf, dtype=torch.float16, device=gpu)
        c.appendQuantized((w, s, s), (w, s, s), seq_ids=[3])
    else:
        c.append(bad[:1, :, :1].contiguous(), bad[:1, :, :1].contiguous(), seq_ids=[3])
    c.append(*want, seq_ids=[3])
    for window in (99, 50, 1):
        got = c.decodeDense(q[3:4].contiguous(), SCALE, window=window, seq_ids=[3])
        _check(got, _reference(c, q[3:4], ids=[3], window=window), dtype, f"window {window}")
    assert c.decodeDense(q[3:4].contiguous(), SCALE, window=100, seq_ids=[3]).isnan().any()
    # (the others are as they were)
    got = c.decodeDense(q, SCALE)
    keep = [0, 1, 2, 4]
    _check(got[keep], _reference(c, q[keep], ids=keep), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_extreme_scores(gpu, dtype):
    """Scores that grow along the sequence, that fall, that are all equal, and
    differences far past what a weight can hold."""
    import torch
    T = 1500
    for case in ("up", "down", "equal", "spike", "huge"):
        c = _cache([T], 8, 2, 64, dtype)
        k = torch.zeros((1, 2, T, D), device=gpu)
        ramp = torch.arange(T, device=gpu).float() / T
        k[..., 0] = {"up": ramp * 400, "down": -ramp * 400, "equal": ramp * 0 + 3,
                     "spike": (torch.arange(T, device=gpu) == 777) * 1000.0,
                     "huge": ramp * 60000}[case]
        v = _randn(gpu, 3, (1, 2, T, D), dtype)
        c.append(k.to(_dt(dtype)), v)
        q = torch.zeros((1, 8, 1, D), device=gpu)
        q[..., 0] = torch.tensor([1.0, 8.0, -1.0, 0.0, 0.5, 30.0, -8.0, 1e-3], device=gpu)[None, :, None]
        q = q.to(_dt(dtype))
        _check(c.decodeDense(q, 1.0), _reference(c, q, scale=1.0), dtype, case)
        _check(c.decodeDense(q, -0.25), _reference(c, q, scale=-0.25), dtype, case + " negative scale")
        _check(c.decodeDense(q, 0.0), _reference(c, q, scale=0.0), dtype, case + " scale 0")


@pytest.mark.parametrize("bits", [4, 8])
def test_quantized_scales(gpu, bits):
    """Scales from 2^-12 to 2^12 (int8: to 2^8, so that their biases, 127.5
    times that, are finite in fp16), in one sequence, and large ones that first
    turn up late."""
    import torch
    T = 900
    for case in ("mixed", "late", "tiny"):
        c = _cache([T], 16, 2, 64, "f16", bits)
        g = torch.Generator(device=gpu).manual_seed(17)
        kw, ks = c.quantizedShapes(1, T)
        w = [torch.randint(-2 ** 31, 2 ** 31, kw, generator=g, device=gpu, dtype=torch.int64).to(torch.int32)
             for _ in range(2)]
        span = {"mixed": torch.rand(ks, generator=g, device=gpu) * 24 - 12,
                "late": torch.where(torch.arange(T, device=gpu)[None, None, :, None] < 700, -8.0, 11.0).expand(ks),
                "tiny": torch.full(ks, -12.0, device=gpu)}[case]
        sign = torch.where(torch.rand(ks, generator=g, device=gpu) < 0.5, -1.0, 1.0)
        if bits == 8:
            span = span.clamp_max(8.0)
        vs = (sign * 2.0 ** span).half()
        vb = (-vs.float() * (2 ** bits - 1) / 2).half()
        ks_ = torch.full(ks, 2.0 ** (-bits), device=gpu).half()
        c.appendQuantized((w[0], ks_, -ks_ * 2 ** (bits - 1)), (w[1], vs, vb))
        q = _randn(gpu, 5, (1, 16, 1, D), "f16")
        want = _reference(c, q)
        got = c.decodeDense(q, SCALE)
        assert want.abs().max() < 60000
        _check(got, want, "f16", case)


def test_steps_and_capture(gpu):
    """A captured [append_step, dense decode] loop against eager calls, with
    the graph replayed between them; two graphs of one cache."""
    import torch
    lens = [3000, 31, 0, 64]
    c = _cache(lens, 32, 8, 64, "bf16", spare=20)
    _fill(gpu, c, lens, 5)
    c.reserve(16, seq_ids=[0, 1, 2, 3])
    q = _randn(gpu, 1, (4, 32, 1, D), "bf16")
    k, v = _randn(gpu, 2, (4, 8, 1, D), "bf16"), _randn(gpu, 3, (4, 8, 1, D), "bf16")
    c.decodeDense(q, SCALE)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for window in (None, 700):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.appendStep(k, v)
            outs.append(c.decodeDense(q, SCALE, window=window))
        graphs.append(graph)
    for step in range(6):
        k.copy_(_randn(gpu, 20 + step, (4, 8, 1, D), "bf16"))
        v.copy_(_randn(gpu, 40 + step, (4, 8, 1, D), "bf16"))
        q.copy_(_randn(gpu, 60 + step, (4, 32, 1, D), "bf16"))
        graphs[step % 2].replay()
        eager = c.decodeDense(q, SCALE, window=(None, 700)[step % 2])
        assert torch.equal(outs[step % 2], eager), f"step {step}"
        other = c.decodeDense(q, SCALE)
        torch.cuda.synchronize()
    c.sync()
    assert [c.seqLen(b) for b in range(4)] == [n + 6 for n in lens]
    _check(other, _reference(c, q), "bf16")


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("lens,Hq,Hkv", [([4700] * 9, 32, 16), ([100 + 131 * i for i in range(40)], 16, 8),
                                         ([700] * 33, 32, 16), ([20000, 3, 900], 8, 8)])
def test_uneven_batches(gpu, dtype, bits, lens, Hq, Hkv):
    """Batches whose parts fit a round of workgroups only with rest, fill
    several, or come one a sequence."""
    log(f"[uneven] {dtype} bits={bits} {len(lens)} of {min(lens)}..{max(lens)} {Hq}/{Hkv}")
    c = _cache(lens, Hq, Hkv, 64, dtype, bits)
    _fill(gpu, c, lens, 17, salient=True)
    q = _randn(gpu, 6, (len(lens), Hq, 1, D), dtype)
    _check(c.decodeDense(q, SCALE), _reference(c, q), dtype)
    some = list(range(len(lens)))[::-1][:7]
    _check(c.decodeDense(q[some].contiguous(), SCALE, seq_ids=some), _reference(c, q[some], ids=some), dtype)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(8, 4), (16, 1)])
def test_replayed_at_other_lengths(gpu, dtype, bits, Hq, Hkv):
    """A graph that was captured over short sequences replays over ones that
    have grown many times over since, in pages taken later, and shrunk."""
    import torch
    log(f"[replay] {dtype} bits={bits} {Hq}/{Hkv}")
    c = _cache([9000] * 4, Hq, Hkv, 64, dtype, bits)
    _fill(gpu, c, [200, 0, 1, 640], 3, salient=True)
    q = _randn(gpu, 4, (4, Hq, 1, D), dtype)
    c.decodeDense(q, SCALE)
    torch.cuda.synchronize()
    graphs = []
    for window in (None, 500):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.decodeDense(q, SCALE, window=window)
        graphs.append((graph, out, window))
    for step, more in enumerate((0, 70, 2000, 6000, -7500, 300)):
        if more > 0:
            n = 4 - step % 2
            k, v = (_randn(gpu, 50 + 2 * step + i, (n, Hkv, more, D), dtype) for i in range(2))
            c.append(k, v, seq_ids=list(range(n)))
        elif more < 0:
            c.trim(-more, seq_ids=[0, 1, 2, 3])
        for graph, out, window in graphs:
            graph.replay()
            _check(out, _reference(c, q, window=window), dtype, f"step {step} window {window}")


def test_streams_rows_and_repeats(gpu):
    """Many rows; other streams at once on their own caches; the same bits
    every time."""
    import torch
    lens = [(37 * i) % 300 for i in range(150)]
    c = _cache(lens, 8, 2, 32, "f16")
    _fill(gpu, c, lens, 5)
    q = _randn(gpu, 1, (150, 8, 1, D), "f16")
    whole = c.decodeDense(q, SCALE)
    _check(whole, _reference(c, q), "f16")
    ids = [140, 3, 77]
    part = c.decodeDense(q[ids].contiguous(), SCALE, seq_ids=ids)
    _check(part, _reference(c, q[ids], ids=ids), "f16")
    caches = []
    for i in range(6):
        ci = _cache([20000], 32, 8, 64, "bf16")
        _fill(gpu, ci, [20000], 50 + i)
        qi = _randn(gpu, 90 + i, (1, 32, 1, D), "bf16")
        caches.append((ci, qi, ci.decodeDense(qi, SCALE)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    for n in range(8):
        got = []
        for i, (ci, qi, _) in enumerate(caches):
            with torch.cuda.stream(streams[(i + n) % 6]):
                got.append(ci.decodeDense(qi, SCALE))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b[2]) for a, b in zip(got, caches)), f"round {n}"


def test_profile_and_prefill_agree(gpu):
    """Timed launches, and the prompt kernel's answer for a single query."""
    import torch
    from bsattn import _lib
    c = _cache([9000], 32, 8, 64, "f16")
    _fill(gpu, c, [9000], 3)
    q = _randn(gpu, 4, (1, 32, 1, D), "f16")
    want = c.decodeDense(q, SCALE)
    c.profile(True)
    assert torch.equal(c.decodeDense(q, SCALE), want)
    ms, n = c.profileRead(_lib.KERNEL_DENSE)
    assert n == 1 and ms > 0
    c.profile(False)
    _check(c.prefill(q, SCALE), _reference(c, q), "f16", "prefill of one token")


def test_refusals(gpu):
    import torch
    import bsattn
    c = _cache([64, 64], 8, 2, 32, "f16")
    _fill(gpu, c, [10, 10], 1)
    q = _randn(gpu, 4, (2, 8, 1, D), "f16")
    for bad in (q.bfloat16(), q[:, :4].contiguous(), q.cpu(), torch.cat([q, q], 2), q.transpose(0, 1)):
        with pytest.raises(ValueError):
            c.decodeDense(bad, SCALE)
    for w in (0, -1):
        with pytest.raises(ValueError):
            c.decodeDense(q, SCALE, window=w)
    s = torch.zeros(8, device=gpu)
    for bad in (s.half(), s[:4], s.cpu(), torch.zeros(16, device=gpu)[::2]):
        with pytest.raises(ValueError):
            c.decodeDense(q, SCALE, sinks=bad)
    for ids in ([0, 0], [0, 2], [-1, 0]):
        with pytest.raises(bsattn.BsattnError):
            c.decodeDense(q, SCALE, seq_ids=ids)
    odd = torch.zeros(2 * 8 * D + 1, dtype=torch.float16, device=gpu)[1:].view(2, 8, 1, D)
    with pytest.raises(bsattn.BsattnError):
        c.decodeDense(odd, SCALE)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (4, 2), (32, 8), (16, 2), (32, 2)])
def test_joins_agree(gpu, dtype, bits, Hq, Hkv):
    """The same bits call after call, timed or not, for counts of parts from
    one to more than a round of the join's rows."""
    import torch
    log(f"[dense joins] {dtype} bits={bits} {Hq}/{Hkv}")
    lens = [1, 129, 300, 1100, 0, 4200, 33]
    c = _cache(lens, Hq, Hkv, 64, dtype, bits, spare=64)
    _fill(gpu, c, lens, 7)
    sinks = torch.linspace(-1, 3, Hq, device=gpu)
    for step in range(3):
        for ids in ([0], [1, 2], [3], [5], [6, 5], list(range(7)), [4, 5, 3]):
            q = _randn(gpu, 10 * step + len(ids), (len(ids), Hq, 1, D), dtype)
            for kw in (dict(), dict(sinks=sinks), dict(window=1000)):
                got = [c.decodeDense(q, SCALE, seq_ids=ids, **kw) for _ in range(3)]
                c.profile(True)
                want = c.decodeDense(q, SCALE, seq_ids=ids, **kw)
                c.profile(False)
                assert all(torch.equal(g, want) for g in got), f"{ids} {kw}"
            _check(got[0], _reference(c, q, ids=ids, window=1000), dtype, f"{ids}")
        k = _randn(gpu, 90 + step, (7, Hkv, 17, D), "f16" if bits else dtype)
        c.append(k, k)
