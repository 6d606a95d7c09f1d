"""Rotary positions (bsattn_rotate) and the norms before them
(bsattn_norm_rotate) against the formulas in 64 bits: layouts, parts of the
head, strides, positions given and taken from the cache, streams, capture and
refusals."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from common import log

pytestmark = pytest.mark.gpu

EPS = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7}  # torch.finfo(t).eps
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest step


def _dt(name):
    import torch
    return torch.float16 if name == "f16" else torch.bfloat16


def _cache(gpu, dtype, Hq=8, Hkv=2, rows=4, blocks=8):
    import bsattn
    return bsattn.BlockSparseKVCache(max_seqs=rows, num_q_heads=Hq, num_kv_heads=Hkv, block_size=32,
                                     dtype=_dt(dtype), top_k=2, max_blocks_per_seq=blocks, device=0)


def _randn(gpu, seed, shape, dtype, scale=1.0):
    import torch
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(_dt(dtype)).to(gpu)


def _reference(x, pos, theta, m, R, interleaved):
    """x [B, H, L, 128] float64, pos [B, L]: (rotated, |a| + |b| of each dim's pair)."""
    phi = pos.astype(np.longdouble)[:, None, :, None] * np.asarray(theta, np.longdouble)
    c, s = np.cos(phi).astype(np.float64) * m, np.sin(phi).astype(np.float64) * m
    y, size = x.copy(), np.abs(x)
    ia = np.arange(0, R, 2) if interleaved else np.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = abs(m) * (np.abs(a) + np.abs(b))
    return y, size


def _check(got, want, size, dtype, steps):
    """One rounding to the output's type (eps / 2 of the value), and `steps`
    fp32 roundings of 2^-24 of the pair's size on the way to it."""
    err = np.abs(got.double().cpu().numpy() - want)
    tol = EPS[dtype] / 2 * (np.abs(want) + steps * 2.0 ** -24 * size) + steps * 2.0 ** -24 * size + TINY[dtype]
    assert (err <= tol).all(), f"error {err.max():.3g}, {(err / tol).max():.3g} of the tolerance"


# Steps of the rotation: the angle in half turns is rounded once (2^-25 of at
# most 1, times pi: 1.6 * 2^-24), cosine and sine to 2 units in the last place
# (4 * 2^-24 of at most 1), their product with m (1) and the two products and
# the sum (2): 9 for each of a and b.  The norm adds the sum of 128 squares (at
# most 8 + 4 + 1 additions deep: 13 / 2 after the root), its mean and eps (1),
# the root (2), offset + weight (1) and two products (2): 13 more.
ROTATE, NORM = 9, 22


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R,interleaved", [(128, False), (128, True), (64, False), (64, True), (96, False),
                                           (20, False), (20, True), (2, False), (2, True), (126, False)])
@pytest.mark.parametrize("B,H,L", [(1, 1, 1), (3, 5, 17), (2, 8, 33)])
def test_rotate(gpu, dtype, R, interleaved, B, H, L):
    import torch
    import bsattn
    log(f"[rotate] {dtype} R={R} interleaved={interleaved} {B}x{H}x{L}")
    c = _cache(gpu, dtype)
    m = 1.0 if R == 64 else 1.1386
    theta = [10000.0 ** (-2.0 * i / R) for i in range(R // 2)]
    rope = bsattn.RoPE(R, interleaved, theta=theta, factor=m)
    m = float(np.float32(m))
    x = _randn(gpu, R + L, (B, H, L, 128), dtype)
    pos = torch.arange(L, dtype=torch.int32)[None] + torch.tensor([[0], [4095], [1 << 24]], dtype=torch.int32)[:B]
    want, size = _reference(x.double().cpu().numpy(), pos.numpy(), theta, m, R, interleaved)
    got = bsattn.applyRotaryPosition(rope, x, c, positions=pos.to(gpu))
    _check(got, want, size, dtype, ROTATE)
    if R < 128:
        assert torch.equal(got[..., R:], x[..., R:])
    # a view into a fused projection [B, L, heads, D]
    p = _randn(gpu, R + L + 1, (B, L, H + 3, 128), dtype)
    p[:, :, 1:1 + H] = x.transpose(1, 2)
    view = p.transpose(1, 2)[:, 1:1 + H]
    assert torch.equal(bsattn.applyRotaryPosition(rope, view, c, positions=pos.to(gpu)), got)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (64, 4), (2, 1), (16, 16)])
@pytest.mark.parametrize("R,interleaved,offset,L", [(128, False, 0.0, 1), (128, False, 1.0, 19), (128, True, 0.0, 5),
                                                    (64, False, 0.0, 16), (96, True, 1.0, 3), (96, False, 0.0, 18),
                                                    (20, False, 1.0, 7), (126, False, 0.0, 3), (2, True, 1.0, 4)])
def test_norm_rotate(gpu, dtype, Hq, Hkv, R, interleaved, offset, L):
    import torch
    import bsattn
    log(f"[norm rotate] {dtype} {Hq}/{Hkv} R={R} interleaved={interleaved} offset={offset} L={L}")
    B, eps = 3, 1e-6
    c = _cache(gpu, dtype, Hq, Hkv)
    rope = bsattn.RoPE(R, interleaved, base=500000.0)
    theta = rope.theta.cpu().numpy()
    p = _randn(gpu, 31 * R + L, (B, L, Hq + 2 * Hkv, 128), dtype, 3.0)
    q, k = p.transpose(1, 2)[:, :Hq], p.transpose(1, 2)[:, Hq:Hq + Hkv]
    w = [_randn(gpu, 5 + i, (128,), dtype) for i in range(2)]
    pos = torch.tensor([[7], [70000], [1 << 20]], dtype=torch.int32) + torch.arange(L, dtype=torch.int32)
    got = c.normRotate(q, k, w[0], w[1], eps, rope, positions=pos.to(gpu), weightOffset=offset)
    for g, x, wi in zip(got, (q, k), w):
        x = x.double().cpu().numpy()
        e = float(np.float32(eps))
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + e) * (wi.double().cpu().numpy() + offset)
        want, size = _reference(y, pos.numpy(), theta, 1.0, R, interleaved)
        # (a weight near -offset: offset + w is rounded to 2^-24 of the larger)
        y1 = np.abs(x) / np.sqrt((x * x).mean(-1, keepdims=True) + e) * (np.abs(wi.double().cpu().numpy()) + offset)
        size = _reference(y1, pos.numpy(), theta, 1.0, R, interleaved)[1]
        assert g.is_contiguous()
        _check(g, want, size, dtype, NORM)


def test_rows_stay_apart(gpu):
    """Zeros, infinities and NaN reach their own head only; a head of zeros
    stays zero under the norm."""
    import torch
    import bsattn
    c = _cache(gpu, "f16")
    rope = bsattn.RoPE(64)
    q, k = _randn(gpu, 1, (1, 8, 6, 128), "f16"), _randn(gpu, 2, (1, 2, 6, 128), "f16")
    w = _randn(gpu, 3, (128,), "f16")
    ref = c.normRotate(q, k, w, w, 1e-5, rope)
    q2, k2 = q.clone(), k.clone()
    q2[0, 3, 2] = 0.0
    q2[0, 4, 1, 77] = math.nan
    k2[0, 1, 5, 0] = math.inf
    got = c.normRotate(q2, k2, w, w, 1e-5, rope)
    assert (got[0][0, 3, 2] == 0).all() and got[0][0, 4, 1].isnan().all() and got[1][0, 1, 5, 0].isnan()
    for g, r, rows in ((got[0], ref[0], [(3, 2), (4, 1)]), (got[1], ref[1], [(1, 5)])):
        keep = torch.ones(g.shape[1:3], dtype=torch.bool)
        for h, t in rows:
            keep[h, t] = False
        assert torch.equal(g[0][keep], r[0][keep])


def test_large_squares(gpu):
    """The norm takes a power of two out of a head, as far as the squares stay
    in fp32's range."""
    import torch
    import bsattn
    c = _cache(gpu, "bf16")
    rope = bsattn.RoPE(128)
    q, k = _randn(gpu, 1, (1, 8, 2, 128), "bf16"), _randn(gpu, 2, (1, 2, 2, 128), "bf16")
    w = _randn(gpu, 3, (128,), "bf16")
    zero = torch.zeros((1, 2), dtype=torch.int32, device=gpu)
    a = c.normRotate(q, k, w, w, 0.0, rope, positions=zero)
    b = c.normRotate(q * 2.0 ** 55, k * 2.0 ** -55, w, w, 0.0, rope, positions=zero)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_positions_from_the_cache(gpu):
    """Without positions the tokens follow those that each row holds, also
    after device-side appends and inside a captured step."""
    import torch
    import bsattn
    dtype = "bf16"
    c = _cache(gpu, dtype, rows=5)
    lens = [0, 31, 32, 77, 5]
    for s, n in enumerate(lens):
        if n:
            c.append(_randn(gpu, s, (1, 2, n, 128), dtype), _randn(gpu, s + 9, (1, 2, n, 128), dtype), seq_ids=[s])
    rope = bsattn.RoPE(128)
    w = _randn(gpu, 3, (128,), dtype)
    ids = [3, 0, 4, 1]

    def explicit(q, k, lens):
        L = q.shape[2]
        pos = torch.tensor([[lens[s] + i for i in range(L)] for s in ids], dtype=torch.int32, device=gpu)
        return (*c.normRotate(q, k, w, w, 1e-6, rope, positions=pos, seq_ids=ids),
                bsattn.applyRotaryPosition(rope, q, c, positions=pos, seq_ids=ids))

    for L in (1, 4, 20):
        q, k = _randn(gpu, L, (4, 8, L, 128), dtype), _randn(gpu, L + 1, (4, 2, L, 128), dtype)
        got = (*c.normRotate(q, k, w, w, 1e-6, rope, seq_ids=ids), bsattn.applyRotaryPosition(rope, q, c, seq_ids=ids))
        for a, b in zip(got, explicit(q, k, lens)):
            assert torch.equal(a, b)
    # a captured step rotates, appends and decodes at the lengths of each replay
    c.reserve(6, seq_ids=ids)
    q, k, v = (_randn(gpu, 60 + i, (4, h, 1, 128), dtype) for i, h in enumerate((8, 2, 2)))
    c.normRotate(q, k, w, w, 1e-6, rope, seq_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, kr = c.normRotate(q, k, w, w, 1e-6, rope, seq_ids=ids)
        c.appendStep(kr, v, seq_ids=ids)
        out = c.decode(qr, 128 ** -0.5, seq_ids=ids)
    now = dict(enumerate(lens))
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = explicit(q, k, now)
        assert torch.equal(qr, want[0]) and torch.equal(kr, want[1]), f"replay {step}"
        for s in ids:
            now[s] += 1
        assert torch.equal(out, c.decode(qr, 128 ** -0.5, seq_ids=ids))
    c.sync()
    assert [c.seqLen(s) for s in range(5)] == [now[s] for s in range(5)]


def test_many_rows_and_streams(gpu):
    """More sequences than a launch takes; another stream; the current device
    stays as it was."""
    import torch
    import bsattn
    c = _cache(gpu, "f16", rows=150, blocks=1)
    rope = bsattn.RoPE(128)
    q = _randn(gpu, 1, (150, 8, 2, 128), "f16")
    pos = (torch.arange(300, dtype=torch.int32, device=gpu) * 37).reshape(150, 2)
    whole = bsattn.applyRotaryPosition(rope, q, c, positions=pos)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        other = bsattn.applyRotaryPosition(rope, q, c, positions=pos)
    st.synchronize()
    assert torch.equal(whole, other) and torch.cuda.current_device() == 0
    for i in (0, 63, 64, 149):
        one = bsattn.applyRotaryPosition(rope, q[i:i + 1].contiguous(), c, positions=pos[i:i + 1].contiguous())
        assert torch.equal(whole[i:i + 1], one)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R,interleaved", [(64, False), (64, True), (20, False), (20, True), (96, False)])
def test_dims_that_stay(gpu, dtype, R, interleaved):
    """Dims past the rotated ones come through bit for bit, infinities, the
    smallest and largest numbers and -0 among them, and touch no other dim."""
    import torch
    import bsattn
    c = _cache(gpu, dtype)
    rope = bsattn.RoPE(R, interleaved, factor=1.25)
    x = _randn(gpu, R, (2, 8, 19, 128), dtype)
    plain = bsattn.applyRotaryPosition(rope, x, c)
    f = torch.finfo(_dt(dtype))
    odd = torch.tensor([math.inf, -math.inf, f.max, f.min, f.tiny, -0.0, 2.0 ** (-24 if dtype == "f16" else -133)],
                       device=gpu).to(_dt(dtype))
    x[..., R:R + 7] = odd
    x[..., 121:] = odd
    got = bsattn.applyRotaryPosition(rope, x, c)
    assert torch.equal(got[..., :R], plain[..., :R])
    assert torch.equal(got[..., R:].view(torch.int16), x[..., R:].view(torch.int16))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R,interleaved", [(128, False), (64, False), (128, True), (20, False)])
def test_large_inputs(gpu, dtype, R, interleaved):
    """More than the caches hold at once: what the rows give on their own."""
    import torch
    import bsattn
    log(f"[large] {dtype} R={R} interleaved={interleaved}")
    B, L, Hq, Hkv = 9, 1301, 32, 4
    c = _cache(gpu, dtype, Hq, Hkv, rows=B)
    rope = bsattn.RoPE(R, interleaved)
    g = torch.Generator(device=gpu).manual_seed(R)
    p = torch.randn((B, L, Hq + Hkv, 128), generator=g, device=gpu).to(_dt(dtype))
    q, k = p.transpose(1, 2)[:, :Hq], p.transpose(1, 2)[:, Hq:]
    assert p.numel() * 2 > 96 << 20
    w = [_randn(gpu, 5 + i, (128,), dtype) for i in range(2)]
    pos = torch.arange(B * L, dtype=torch.int32, device=gpu).reshape(B, L)
    alone = bsattn.applyRotaryPosition(rope, p.transpose(1, 2), c, positions=pos)
    whole = c.normRotate(q, k, w[0], w[1], 1e-6, rope, positions=pos)
    for b in (0, 4, 8):
        one = pos[b:b + 1].contiguous()
        assert torch.equal(alone[b:b + 1], bsattn.applyRotaryPosition(rope, p[b:b + 1].transpose(1, 2), c, positions=one))
        part = c.normRotate(q[b:b + 1], k[b:b + 1], w[0], w[1], 1e-6, rope, positions=one)
        assert torch.equal(whole[0][b:b + 1], part[0]) and torch.equal(whole[1][b:b + 1], part[1])


def test_offsets_past_32_bits(gpu):
    """A tensor of more than 2^31 elements, whole and through its strides."""
    import torch
    import bsattn
    log("[rotate] 2^31 elements")
    H, L = 64, 270001
    c = _cache(gpu, "bf16")
    rope = bsattn.RoPE(128)
    x = torch.zeros((1, H, L, 128), dtype=torch.bfloat16, device=gpu)
    assert x.numel() > 2 ** 31
    tail = _randn(gpu, 1, (1, H, 21, 128), "bf16")
    x[:, :, -21:] = tail
    pos = torch.arange(L, dtype=torch.int32, device=gpu)[None]
    want = bsattn.applyRotaryPosition(rope, tail, c, positions=pos[:, -21:].contiguous())
    got = bsattn.applyRotaryPosition(rope, x, c, positions=pos)
    assert torch.equal(got[:, :, -21:], want) and not got[:, :, :-21].any()
    view = x.view(1, L, H, 128).transpose(1, 2)  # the same memory, tokens first
    assert torch.equal(bsattn.applyRotaryPosition(rope, view[:, :, -3:], c, positions=pos[:, -3:].contiguous()),
                       bsattn.applyRotaryPosition(rope, view[:, :, -3:].contiguous(), c, positions=pos[:, -3:].contiguous()))


def test_in_place(gpu):
    import torch
    import bsattn
    from bsattn import _lib
    for R, inter in ((128, False), (96, False), (64, True)):
        c = _cache(gpu, "bf16")
        rope = bsattn.RoPE(R, inter)
        q = _randn(gpu, 1, (2, 8, 21, 128), "bf16")
        want = bsattn.applyRotaryPosition(rope, q, c)
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(_lib.lib().bsattn_rotate(c._h, rope._ref, q.data_ptr(), None, 8, None, 2, 21, None, q.data_ptr(),
                                            stream))
        assert torch.equal(q, want)
        # not from a view
        st = (ctypes.c_int64 * 3)(8 * 21 * 128, 128, 8 * 128)
        rc = _lib.lib().bsattn_rotate(c._h, rope._ref, q.data_ptr(), st, 8, None, 2, 21, None, q.data_ptr(), stream)
        assert rc == _lib.ERR_INVALID


def test_profile(gpu):
    import bsattn
    from bsattn import _lib
    c = _cache(gpu, "f16")
    rope = bsattn.RoPE(128)
    c.profile(True)
    bsattn.applyRotaryPosition(rope, _randn(gpu, 1, (2, 8, 3, 128), "f16"), c)
    ms, n = c.profileRead(_lib.KERNEL_ROTATE)
    assert n == 1 and ms > 0


def test_refusals(gpu):
    import torch
    import bsattn
    c = _cache(gpu, "f16")
    rope = bsattn.RoPE(128)
    q, k = _randn(gpu, 1, (2, 8, 4, 128), "f16"), _randn(gpu, 2, (2, 2, 4, 128), "f16")
    w = _randn(gpu, 3, (128,), "f16")
    pos = torch.zeros((2, 4), dtype=torch.int32, device=gpu)
    bad_q = [q.bfloat16(), q.cpu(), q[..., :64], q[:, :4], torch.zeros(2, 8, 4, 256, dtype=q.dtype, device=gpu)[..., ::2],
             torch.zeros(2 * 8 * 4 * 128 + 1, dtype=q.dtype, device=gpu)[1:].view(2, 8, 4, 128), q[:, :, :0], q[0],
             torch.zeros(2, 8, 4, 132, dtype=q.dtype, device=gpu)[..., :128]]
    for x in bad_q:
        with pytest.raises(ValueError):
            c.normRotate(x, k, w, w, 1e-6, rope, positions=pos)
    for x in bad_q[:3] + bad_q[4:]:
        with pytest.raises(ValueError):
            bsattn.applyRotaryPosition(rope, x, c, positions=pos)
    for p in (pos.long(), pos.cpu(), pos[:, :3].contiguous(), pos.t().contiguous(), pos[:1]):
        with pytest.raises(ValueError):
            bsattn.applyRotaryPosition(rope, q, c, positions=p)
    for bw in (w.float(), w[:64], w.cpu()):
        with pytest.raises(ValueError):
            c.normRotate(q, k, bw, w, 1e-6, rope)
        with pytest.raises(ValueError):
            c.normRotate(q, k, w, bw, 1e-6, rope)
    with pytest.raises(ValueError):
        c.normRotate(q, k[:1], w, w, 1e-6, rope)
    for kw in (dict(eps=-1.0), dict(eps=math.nan), dict(eps=1e-6, weightOffset=math.inf)):
        with pytest.raises(bsattn.BsattnError):
            c.normRotate(q, k, w, w, rope=rope, **kw)
    for ids in ([0, 0], [0, 4], [-1, 0]):
        with pytest.raises(bsattn.BsattnError):
            bsattn.applyRotaryPosition(rope, q, c, seq_ids=ids)
