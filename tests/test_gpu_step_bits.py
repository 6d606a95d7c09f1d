"""Tree attention holds values exactly and weights in 16 bits, however many
columns a launch has: tokens whose small values have all the weight, and pairs
of tokens whose values nearly cancel."""
from __future__ import annotations

import pytest

from common import log
from test_gpu_dense import D, HALF_STEP, SCALE, _cache, _dt, _held, _randn
from test_gpu_step import _rows, _step, _tree

pytestmark = pytest.mark.gpu

# (Hq, Hkv, cached tokens, nodes): 16, 32, 64, 128 and 256 columns a workgroup, those of 64 and 128 in waves of one
# and (long sequences) of two column tiles
WIDTHS = [(8, 2, 700, 4), (8, 2, 700, 8), (32, 8, 700, 16), (32, 8, 700, 32), (32, 8, 20000, 16), (32, 8, 20000, 32),
          (16, 1, 700, 64), (16, 1, 700, 19)]


def _attend(gpu, dtype, keys, values, q, N):
    """Outputs [N, Hq, D] of a tree behind keys / values [Hkv, T, D]; the new tokens' keys are zero."""
    Hkv, T = keys.shape[:2]
    c = _cache([T], q.shape[1], Hkv, 64, dtype, spare=64)
    c.append(keys[None].contiguous(), values[None].contiguous())
    step = _step(gpu, [c], [N], [_tree(3, N)])
    _, k, v = _rows(gpu, c, 8, N, fused=False)
    c.appendPacked(k.zero_(), v, step)
    return c.attendTree(q, step, SCALE)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,T,N", WIDTHS)
def test_small_values_of_the_heaviest_token(gpu, dtype, Hq, Hkv, T, N):
    """One token has all the weight, and values of 2^-8 to 2^-30 (fp16: its least, 2^-24) beside others of 1: the
    outputs are its values, which the type holds, and nothing is rounded."""
    import torch
    log(f"[heaviest] {dtype} {Hq}/{Hkv} T={T} N={N}")
    at = 261
    keys, values = (_randn(gpu, 3 + x, (Hkv, T, D), dtype) for x in (0, 1))
    # its score is 181 where the others' deviate by 8: their weights add to less than 2^-150
    keys[:, at] = 2.0
    d = torch.arange(D, device=gpu)
    small = (1 + (d * 37 % 128) / 128) * 2.0 ** -(8 + d % (23 if dtype == "bf16" else 17)) * (1 - 2 * (d % 2))
    values[:, at] = small.to(_dt(dtype))
    q = torch.full((N, Hq, D), 8.0, dtype=_dt(dtype), device=gpu)
    out = _attend(gpu, dtype, keys, values, q, N)
    want = values[:, at].repeat_interleave(Hq // Hkv, 0).expand(N, Hq, D)
    wrong = (out != want).nonzero()
    assert not len(wrong), (len(wrong), out[tuple(wrong[0])].item(), want[tuple(wrong[0])].item())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,T,N", WIDTHS)
def test_weights_of_16_bits(gpu, dtype, Hq, Hkv, T, N):
    """Two tokens of a unit share the weight, about 1 : 0.7, and values of -1 : 1.42 nearly cancel.  Weights are held to
    2^-16, their sum as well.  Scores are single products, of 70 at most as powers of two: three roundings of 2^-24 each
    move a weight by 2^-16 x 0.61.  The other tokens' weights are e^-42 of these.  So an output is off by 2^-16 (2 + 2 x 0.61) < 2^-14 of the sum
    of its terms' magnitudes, and by its own rounding."""
    import torch
    log(f"[weights] {dtype} {Hq}/{Hkv} T={T} N={N}")
    keys, values = torch.zeros((Hkv, T, D), dtype=_dt(dtype), device=gpu), _randn(gpu, 4, (Hkv, T, D), dtype)
    a, b = 130, 141
    keys[:, a, 0], keys[:, b, 0] = 8.0, 7.9375
    d = torch.arange(D, device=gpu)
    values[:, a] = (1 + d / 128).to(_dt(dtype))
    values[:, b] = (-(1 + d / 128) * 1.42 * (1 + ((d * 29) % 64 - 32) / 512)).to(_dt(dtype))
    q = torch.zeros((N, Hq, D), dtype=_dt(dtype), device=gpu)
    g = torch.Generator(device=gpu).manual_seed(7)
    q[..., 0] = (60 + 8 * torch.rand((N, Hq), device=gpu, generator=g)).to(_dt(dtype))
    out = _attend(gpu, dtype, keys, values, q, N).double()
    s = q[..., :1].double() * SCALE * torch.tensor([8.0, 7.9375], dtype=torch.float64, device=gpu)
    p = torch.softmax(s, -1)
    pair = values[:, [a, b]].double().repeat_interleave(Hq // Hkv, 0)  # [Hq, 2, D]
    terms = p[..., None] * pair[None]
    want, reach = terms.sum(2), terms.abs().sum(2)
    err = (out - want).abs() / (HALF_STEP[dtype] * want.abs() + 2.0 ** -14 * reach)
    assert err.max().item() <= 1, err.max().item()
