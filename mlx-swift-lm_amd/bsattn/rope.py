"""Rotary positions: RoPE, initializeRope and applyRotaryPosition.

Mirrors Libraries/MLXLMCommon/RoPEApplication.swift:23-27 and the variants
that Libraries/MLXLMCommon/RoPEUtils.swift:210 chooses from a model's
rope_scaling entry.  Every variant is a table of angles per position (64-bit)
and a factor on the rotated dims, computed once here; the kernels take both.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check
from .cache import BlockSparseKVCache, _row_ids, _stream

HEAD_DIM = 128


class RoPE:
    """Rotary positions of the first `dims` dims of each head: pair i turns by
    `scale * base^(-2i / dims)` radians per position, or by theta[i];
    traditional: pairs are neighbours (2i, 2i + 1), otherwise (i, i + dims / 2);
    factor multiplies the rotated dims.  Keep the object while calls or graphs
    that use it are pending."""

    def __init__(self, dims: int, traditional: bool = False, base: float = 10000.0, scale: float = 1.0, *,
                 theta: Optional[Sequence[float]] = None, factor: float = 1.0, device: int | torch.device = 0):
        if dims < 2 or dims > HEAD_DIM or dims % 2:
            raise ValueError(f"rope dims must be even, from 2 to {HEAD_DIM} (got {dims})")
        if theta is None:
            if not base > 0.0:
                raise ValueError(f"rope base must be positive (got {base})")
            theta = [scale * base ** (-2.0 * i / dims) for i in range(dims // 2)]
        theta = [float(t) for t in theta]
        if len(theta) != dims // 2:
            raise ValueError(f"rope theta must hold {dims // 2} angles (got {len(theta)})")
        if not all(math.isfinite(t) for t in theta) or not math.isfinite(factor):
            raise ValueError("rope angles and factor must be finite")
        self.device = torch.device("cuda", device if isinstance(device, int) else device.index or 0)
        self.index = self.device.index
        self.dims, self.traditional, self.factor = dims, bool(traditional), float(factor)
        self.theta = torch.tensor(theta, dtype=torch.float64, device=self.device)
        # (the table is ready before any stream uses it)
        torch.cuda.current_stream(self.device).synchronize()
        self._c = _lib.Rope(theta=self.theta.data_ptr(), dims=dims, interleaved=int(self.traditional),
                            factor=self.factor, reserved=0)
        self._ref = ctypes.byref(self._c)


def _positive(config: dict, key: str, default=None) -> float:
    v = config.get(key, default)
    if v is None:
        raise ValueError(f"rope scaling needs {key}")
    v = float(v)
    if not (math.isfinite(v) and v > 0.0):
        raise ValueError(f"rope scaling {key} must be positive (got {v})")
    return v


def ropeAngles(dims: int, base: float, scalingConfig: Optional[dict] = None,
               maxPositionEmbeddings: Optional[int] = None):
    """(angles per position, factor on the rotated dims) of a model
    configuration: rope_theta, rope_scaling and max_position_embeddings.

    linear: every angle / factor.  llama3 (Llama3RoPE): pairs that turn less
    than low_freq_factor times in the original context are divided by factor,
    those above high_freq_factor stay, linear in the turns between.  yarn
    (YarnRoPE): divided by factor past the pair that turns beta_slow times,
    kept up to the one that turns beta_fast times, linear in the pair's index
    between; dims scaled by (0.1 mscale ln factor + 1) / (0.1 mscale_all_dim ln
    factor + 1).  longrope / su (SuScaledRoPE): each divided by its long_factor;
    dims scaled by sqrt(1 + ln(extension) / ln(original context))."""
    if not base > 0.0:
        raise ValueError(f"rope base must be positive (got {base})")
    theta = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scalingConfig is None:
        return theta, 1.0
    kind = scalingConfig.get("rope_type", scalingConfig.get("type", "default"))
    if kind in ("default", "mrope"):
        return theta, 1.0
    if kind == "linear":
        f = _positive(scalingConfig, "factor")
        return [t / f for t in theta], 1.0
    if kind == "llama3":
        f = _positive(scalingConfig, "factor")
        lo, hi = _positive(scalingConfig, "low_freq_factor", 1.0), _positive(scalingConfig, "high_freq_factor", 4.0)
        first = _positive(scalingConfig, "original_max_position_embeddings", 8192)
        if hi <= lo:
            raise ValueError("rope scaling high_freq_factor must exceed low_freq_factor")
        out = []
        for t in theta:
            turns = first * t / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            out.append(keep * t + (1.0 - keep) * t / f)
        return out, 1.0
    if kind == "yarn":
        f = _positive(scalingConfig, "factor")
        first = _positive(scalingConfig, "original_max_position_embeddings", 4096)
        edges = [dims * math.log(first / (_positive(scalingConfig, key, default) * 2.0 * math.pi)) /
                 (2.0 * math.log(base)) for key, default in (("beta_fast", 32.0), ("beta_slow", 1.0))]
        lo, hi = max(math.floor(edges[0]), 0), min(math.ceil(edges[1]), dims - 1)
        span = hi - lo if hi != lo else 0.001
        out = []
        for i, t in enumerate(theta):
            ramp = min(1.0, max(0.0, (i - lo) / span))
            out.append(t * (1.0 - ramp) + t / f * ramp)

        def mscale(m):
            return 1.0 if f <= 1.0 else 0.1 * m * math.log(f) + 1.0
        return out, mscale(float(scalingConfig.get("mscale", 1.0))) / mscale(float(scalingConfig.get("mscale_all_dim", 0.0)))
    if kind in ("longrope", "su"):
        first = _positive(scalingConfig, "original_max_position_embeddings", 4096)
        factors = scalingConfig.get("long_factor")
        if factors is None:
            raise ValueError("rope scaling needs long_factor")
        if isinstance(factors, (int, float)):
            factors = [factors] * (dims // 2)
        if len(factors) != dims // 2 or not all(float(x) > 0.0 for x in factors):
            raise ValueError(f"rope scaling long_factor must hold {dims // 2} positive numbers")
        if maxPositionEmbeddings is None:
            raise ValueError("longrope needs maxPositionEmbeddings")
        extension = maxPositionEmbeddings / first
        m = math.sqrt(1.0 + math.log(extension) / math.log(first)) if extension > 1.0 else 1.0
        return [t / float(x) for t, x in zip(theta, factors)], m
    raise ValueError(f"rope scaling type {kind!r} is not supported")


def initializeRope(dims: int, base: float, traditional: bool, scalingConfig: Optional[dict] = None,
                   maxPositionEmbeddings: Optional[int] = None, device: int | torch.device = 0) -> RoPE:
    """The RoPE of a model configuration (initializeRope, RoPEUtils.swift:210)."""
    if dims < 2 or dims > HEAD_DIM or dims % 2:
        raise ValueError(f"rope dims must be even, from 2 to {HEAD_DIM} (got {dims})")
    theta, factor = ropeAngles(dims, base, scalingConfig, maxPositionEmbeddings)
    return RoPE(dims, traditional, theta=theta, factor=factor, device=device)


def applyRotaryPosition(rope: RoPE, x: torch.Tensor, cache: BlockSparseKVCache,
                        positions: Optional[torch.Tensor] = None,
                        seq_ids: Optional[Sequence[int]] = None) -> torch.Tensor:
    """x [B, H, L, 128] (a view whose heads are contiguous will do) with its
    positions rotated in, as a dense tensor.  positions [B, L] int32; by
    default each sequence's tokens follow those that the cache holds (rotate,
    then append)."""
    strides, (B, heads, L, _) = cache._check_strided(x, "x")
    cache._check_rope(rope)
    pos = cache._check_positions(positions, B, L)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    check(cache._lib.bsattn_rotate(cache._h, rope._ref, x.data_ptr(), strides, heads, _row_ids(seq_ids, B), B, L, pos,
                                   out.data_ptr(), _stream(cache.device)))
    return out


__all__ = ["RoPE", "ropeAngles", "initializeRope", "applyRotaryPosition"]
