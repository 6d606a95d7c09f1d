"""Angles of the rotary variants (bsattn.rope.ropeAngles) against their
definitions written with numpy, and what is refused.  CPU only."""
from __future__ import annotations

import math

import numpy as np
import pytest

from bsattn.rope import RoPE, initializeRope, ropeAngles


def _turning(R, base):
    return np.exp(-np.arange(R // 2) * (2.0 / R) * np.log(base))


def _close(got, want):
    # a power, a product and a quotient in 64 bits: a few roundings of 2^-53
    # each; the two sides take the power in different ways (an exponent of at
    # most 14 costs exp 14 * 2^-53)
    np.testing.assert_allclose(np.asarray(got), want, rtol=64 * 2.0 ** -53, atol=0)


@pytest.mark.parametrize("R", [2, 20, 64, 96, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1e6])
def test_plain_and_linear(R, base):
    theta, m = ropeAngles(R, base)
    _close(theta, _turning(R, base))
    assert m == 1.0
    theta, m = ropeAngles(R, base, {"type": "linear", "factor": 8.0})
    _close(theta, _turning(R, base) / 8.0)
    assert m == 1.0
    assert ropeAngles(R, base, {"rope_type": "default"})[1] == 1.0


@pytest.mark.parametrize("R", [64, 128])
def test_llama3(R):
    cfg = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
               original_max_position_embeddings=8192)
    theta, m = ropeAngles(R, 500000.0, cfg)
    t = _turning(R, 500000.0)
    wave = 2 * np.pi / t
    smooth = (8192 / wave - 1.0) / 3.0
    want = np.where(wave < 8192 / 4.0, t, np.where(wave > 8192 / 1.0, t / 8.0, (1 - smooth) * t / 8.0 + smooth * t))
    # the turns' difference from 1 loses at most 4 bits to cancellation here
    np.testing.assert_allclose(theta, want, rtol=1024 * 2.0 ** -53, atol=0)
    assert m == 1.0 and (want < t).any() and (want == t).any()


def test_yarn():
    cfg = dict(type="yarn", factor=4.0, original_max_position_embeddings=32768)
    theta, m = ropeAngles(128, 1e6, cfg)
    t = _turning(128, 1e6)
    edge = [64 * math.log(32768 / (2 * math.pi * r), 1e6) for r in (32, 1)]
    lo, hi = math.floor(edge[0]), math.ceil(edge[1])
    keep = 1 - np.clip((np.arange(64) - lo) / (hi - lo), 0, 1)
    _close(theta, t / 4.0 * (1 - keep) + t * keep)
    assert m == 0.1 * math.log(4.0) + 1.0
    assert ropeAngles(128, 1e6, dict(cfg, mscale=1.0, mscale_all_dim=1.0))[1] == 1.0


def test_longrope():
    factors = [1.0 + 0.5 * i for i in range(48)]
    cfg = dict(rope_type="longrope", original_max_position_embeddings=4096, long_factor=factors)
    theta, m = ropeAngles(96, 10000.0, cfg, 131072)
    _close(theta, _turning(96, 10000.0) / np.array(factors))
    assert m == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)), rel=1e-15)
    assert ropeAngles(96, 10000.0, cfg, 4096)[1] == 1.0


@pytest.mark.parametrize("call,msg", [
    (lambda: initializeRope(63, 1e4, False), "even"),
    (lambda: initializeRope(0, 1e4, False), "even"),
    (lambda: initializeRope(130, 1e4, False), "even"),
    (lambda: RoPE(130), "even"),
    (lambda: RoPE(64, base=0.0), "base"),
    (lambda: RoPE(64, theta=[1.0]), "32 angles"),
    (lambda: RoPE(2, theta=[math.inf]), "finite"),
    (lambda: ropeAngles(64, -1.0), "base"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "linear"}), "factor"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "linear", "factor": 0.0}), "factor"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "spiral", "factor": 2.0}), "spiral"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "longrope", "long_factor": [1.0]}, 8192), "long_factor"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "longrope"}, 8192), "long_factor"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "longrope", "long_factor": [1.0] * 32}), "maxPositionEmbeddings"),
    (lambda: ropeAngles(64, 1e4, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0,
                                  "high_freq_factor": 4.0}), "high_freq_factor"),
])
def test_refusals(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()
