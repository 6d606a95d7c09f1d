"""Calls at the edges of the operators around the cache: what a refused call
leaves behind, and inputs whose numbers lie far apart."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

D = 128
SCALE = D ** -0.5


def test_a_refused_step_appends_nothing(gpu):
    """Queries that the dense decode cannot read: the step is refused before
    its token is appended, and the same step with readable ones then runs."""
    import torch
    import bsattn
    c = bsattn.BlockSparseKVCache(max_seqs=2, num_q_heads=8, num_kv_heads=2, block_size=32, dtype=torch.float16,
                                  top_k=2, max_blocks_per_seq=4, device=0)
    k = torch.randn((2, 2, 40, D), device=gpu).half()
    c.append(k, k)
    q = torch.randn((2, 8, 1, D), device=gpu).half()
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16, device=gpu)[1:].view_as(q).copy_(q)
    new = torch.randn((2, 2, 1, D), device=gpu).half()
    pages = c.freePages
    for _ in range(2):
        with pytest.raises(ValueError):
            bsattn.attentionWithCacheUpdate(odd, new, new, c, SCALE, dense=True)
    assert [c.seqLen(b) for b in range(2)] == [40, 40] and c.freePages == pages
    got = bsattn.attentionWithCacheUpdate(q, new, new, c, SCALE, dense=True)
    assert [c.seqLen(b) for b in range(2)] == [41, 41]
    assert torch.equal(got, c.decodeDense(q, SCALE))


def _spread(gpu, bits, Hq, Hkv, T, seed):
    """Queries [2, Hq, 1, D] and tokens [2, Hkv, T, D] whose scores differ by
    several units, with nothing but what the caller adds along dim 0: there the
    queries hold 4, so a key of x there adds 4 x SCALE to its scores."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(seed)
    q = 2 * torch.randn((2, Hq, 1, D), generator=g, device=gpu)
    q[..., 0] = 4
    k, v = (torch.randn((2, Hkv, T, D), generator=g, device=gpu) for _ in range(2))
    k[..., 0] = 0
    return q.half(), k, v


def _run(gpu, bits, Hq, Hkv, q, k, v):
    """The dense decode over these tokens and the formula over what the cache
    holds, both [2, Hq, 1, D] and [2, Hq, D]."""
    import torch
    from test_gpu_dense import _cache, _reference
    T = k.shape[2]
    c = _cache([T] * 2, Hq, Hkv, 64, "f16", bits)
    c.append(k.half(), v.half())
    got, want = c.decodeDense(q, SCALE), _reference(c, q)
    assert want.abs().max() < 60000 and torch.equal(got, c.decodeDense(q, SCALE))
    return got, want


# Tolerances of the next tests are those of the dense decode's own, row by row:
# rounding to fp16, and 0.3 of half a step of the row's root mean square for all
# before it.  For N(0, 1) values those are the offset of 1024 that is taken off
# the codes twice a unit of 32 tokens, with roundings of 2^-24 / sqrt 3 of 1024
# sum p s each (s: the scale, 1 / 3.2 of a value's deviation for int4, 1 / 54
# for int8): 0.75 sqrt(2 / 3) 2^-14 32 / 3.2 / sqrt 32 = 2^-13.9 of the output,
# 0.13 of half a step, for equal weights and less for others; and the scores,
# whose offset of 1024 sum q costs each weight up to 2^-14 |sum q| s SCALE
# (|sum q| < 60: 2^-13.3, 0.2 of half a step, and the weights' errors differ).
SHAPES = [(8, 2), (32, 8), (32, 2)]  # groups of 4 and of 16


@pytest.mark.parametrize("bits,out", [(4, 10.0), (8, 200.0)])
@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("T", [300, 2100, 20000])
@pytest.mark.parametrize("score", [3.0, -5.0])
def test_large_scales_of_little_weight(gpu, bits, out, Hq, Hkv, T, score):
    """One token in 32 has values, and so a scale, many times the others', and
    e^-4 or e^-12 of the weight of the largest: the others keep their bits."""
    from test_gpu_dense import _check
    q, k, v = _spread(gpu, bits, Hq, Hkv, T, 100 * bits + T)
    odd = slice(5, None, 32)
    k[:, :, odd, 1:] *= 0.1
    k[:, :, odd, 0] = score / (4 * SCALE)
    v[:, :, odd] *= out
    _check(*_run(gpu, bits, Hq, Hkv, q, k, v), "f16", f"{T} tokens")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("T", [300, 5000])
@pytest.mark.parametrize("half", [0, 1])
def test_large_scales_in_one_half(gpu, bits, Hq, Hkv, T, half):
    """Tokens of large values in dims 0-63 or 64-127 alone, with scores like
    any other's: the other half of the dims keeps its bits."""
    from test_gpu_dense import _check
    q, k, v = _spread(gpu, bits, Hq, Hkv, T, 7 * bits + T + half)
    v[:, :, 3::16, 64 * half:64 * half + 64] *= 1000
    got, want = _run(gpu, bits, Hq, Hkv, q, k, v)
    for i in range(2):
        dims = slice(64 * i, 64 * i + 64)
        _check(got[..., dims], want[..., dims], "f16", f"half {i}")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("times", [30.0, 1000.0, 6000.0])
def test_large_scales_everywhere(gpu, bits, Hq, Hkv, times):
    from test_gpu_dense import _check
    q, k, v = _spread(gpu, bits, Hq, Hkv, 3000, 11 * bits)
    _check(*_run(gpu, bits, Hq, Hkv, q, k, v * times), "f16", f"times {times}")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv", SHAPES)
@pytest.mark.parametrize("slope", [30.0, -30.0])
def test_large_scales_that_lose_their_weight(gpu, bits, Hq, Hkv, slope):
    """Scores that rise along the sequence, from tokens of large values whose
    weight is all there is at first to ones of small values, and the other way
    round."""
    import torch
    from test_gpu_dense import _check
    T = 4000
    q, k, v = _spread(gpu, bits, Hq, Hkv, T, 13 * bits)
    ramp = torch.linspace(0, 1, T, device=gpu)
    # (int4 keys of up to 85 have scales of 6: a small sum of the queries' dims)
    q[..., 1:] *= 0.125
    k *= 0.3
    k[..., 0] = (ramp if slope > 0 else 1 - ramp) * abs(slope) / (4 * SCALE)
    large = torch.where(ramp < 0.3, 500.0, 1.0)
    v *= large[:, None]
    _check(*_run(gpu, bits, Hq, Hkv, q, k, v), "f16", f"slope {slope}")


@pytest.mark.parametrize("dtype,bits", [("bf16", 8), ("f16", 4)])
def test_quantizing_keeps_forks_shared(gpu, dtype, bits):
    """toQuantized of a cache whose sequences share blocks, in a pool that
    holds no more: the same codes as sequence by sequence, as many free pages
    as before, and sequences that are independent from then on."""
    import torch
    from test_gpu_dense import _check, _dt, _randn, _reference
    import bsattn
    geometry = dict(max_seqs=9, num_q_heads=8, num_kv_heads=2, block_size=32, top_k=2, max_blocks_per_seq=40, device=0)
    c = bsattn.BlockSparseKVCache(dtype=_dt(dtype), num_pages=60, **geometry)
    plain = bsattn.BlockSparseKVCache(dtype=torch.float16, kv_bits=bits, **geometry)
    k, v = (_randn(gpu, i, (1, 2, 1010, D), dtype) for i in (1, 2))
    c.append(k, v, seq_ids=[8])
    c.fork([8] * 4, [0, 1, 2, 3], [1010, 992, 500, 31])
    more = _randn(gpu, 3, (1, 2, 70, D), dtype)
    c.append(more, more, seq_ids=[1])
    c.fork([1, 1], [4, 5], [1062, 1000])
    c.append(more, more, seq_ids=[6])
    c.trim(400, seq_ids=[4])
    lens = [c.seqLen(s) for s in range(9)]
    q = c.toQuantized(bits=bits)
    assert [q.seqLen(s) for s in range(9)] == lens and q.freePages == c.freePages
    for s in range(9):
        if lens[s]:
            k, v = c.export([s])
            plain.append(k.half(), v.half(), seq_ids=[s])
            for a, b in zip(sum(q.exportQuantized([s]), ()), sum(plain.exportQuantized([s]), ())):
                assert torch.equal(a, b), f"sequence {s}"
            assert torch.equal(q.exportSummaries(s), plain.exportSummaries(s)), f"sequence {s}"
    new = _randn(gpu, 5, (9, 2, 1, D), "f16")
    for x in (q, plain):
        x.append(new, new)
    x = _randn(gpu, 6, (9, 8, 1, D), "f16")
    assert torch.equal(q.decode(x, SCALE), plain.decode(x, SCALE))
    _check(q.decodeDense(x, SCALE), _reference(plain, x), "f16")
    q.reset(list(range(9)))
    assert q.freePages == 60


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv", SHAPES)
def test_large_scales_of_branches(gpu, bits, Hq, Hkv):
    """Large scales in blocks that branches share and in what they have of
    their own; a window and sinks beside them."""
    import torch
    from test_gpu_dense import _cache, _check, _reference
    q, k, v = _spread(gpu, bits, Hq, Hkv, 2500, 17 * bits)
    v[:, :, 5::32] *= 100
    v[:, :, 9::32, :64] *= 1000
    c = _cache([2600] * 14, Hq, Hkv, 64, "f16", bits)
    c.append(k.half(), v.half(), seq_ids=[0, 1])
    c.fork([0] * 9 + [1] * 3, list(range(2, 14)))
    c.append((k[:1, :, :70] * 1.5).half().expand(12, -1, -1, -1).contiguous(),
             v[:1, :, :70].half().expand(12, -1, -1, -1).contiguous(), seq_ids=list(range(2, 14)))
    q = torch.cat([q[:1] * (1 - 0.05 * i) for i in range(14)]).contiguous()
    sinks = torch.linspace(-2, 6, Hq, device=gpu)
    for kw in (dict(), dict(sinks=sinks), dict(window=900, sinks=sinks)):
        got, want = c.decodeDense(q, SCALE, **kw), _reference(c, q, **kw)
        for i in range(2):
            dims = slice(64 * i, 64 * i + 64)
            _check(got[..., dims], want[..., dims], "f16", f"half {i} {list(kw)}")
