"""attentionWithCacheUpdate for the block-sparse cache.

Mirrors Libraries/MLXLMCommon/AttentionUtils.swift:37-77: the function a
model's attention module calls with freshly projected queries / keys /
values.  The reference routes on the cache's dynamic type; the block-sparse
cache is one more branch that appends the new token(s) and runs the
HIP select + gather-attention path.  Other cache types stay on the
reference's own dense path and are not handled here.
"""
from __future__ import annotations

import torch

from .cache import BlockSparseKVCache


# A pass of up to MAX_QUERIES tokens (the speculative-verify shape, L =
# numDraft + 1) runs block-sparse, each query on its own prefix, so that its
# outputs equal token-by-token decoding; longer passes (prefill chunks) run
# dense causal attention, as the reference computes for L > 1.
MAX_QUERIES = 16


def attentionWithCacheUpdate(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                             cache, scale: float, mask="none", *, dense: bool = False, window=None, sinks=None,
                             rope=None, norms=None, step=None) -> torch.Tensor:
    """queries [B, Hq, L, D], keys / values [B, Hkv, L, D] -> [B, Hq, L, D].

    dense: attention over every token instead of the selected blocks, for
    layers that take no selection; a single token may see the last `window`
    tokens only, and each head a sink logit ([Hq] float32).  rope: queries and
    keys come without positions and get those behind the cached tokens first;
    norms: (qWeight, kWeight, eps) or (qWeight, kWeight, eps, weightOffset) of
    the per-head RMS norms ahead of the rope, in the same pass.  Queries and
    keys may then be views into a fused projection; values are contiguous in any
    case (of a view, the caller makes a copy).

    step: a Step that was mapped for the new tokens.  queries [rows, Hq, D] and
    keys / values [rows, Hkv, D] are its packed rows, with their positions
    (step.positions), all of them views if need be; they are appended and
    attend densely, each to what its request held and to its ancestors (mask
    "none": the step says who sees whom)."""
    if not isinstance(cache, BlockSparseKVCache):
        raise TypeError("attentionWithCacheUpdate here handles BlockSparseKVCache only; "
                        "other caches use the reference's dense path")
    if step is not None:
        if rope is not None or norms is not None or mask not in ("none", None):
            raise ValueError("a step's rows come with their positions, and take no mask")
        # nothing is appended that could not be attended to
        cache._check_packed(queries, "queries", cache._hq, step.rows)
        cache._check_window(window)
        cache._check_sinks(sinks)
        if step.ancestors is None:
            raise ValueError("a step of more than 64 tokens a request can be appended, not attended to")
        cache.appendPacked(keys, values, step)
        return cache.attendTree(queries, step, scale, window=window, sinks=sinks)
    if (window is not None or sinks is not None) and not dense:
        raise ValueError("window and sinks belong to dense attention (dense=True)")
    if norms is not None and rope is None:
        raise ValueError("norms are applied in the rope's pass: give a rope")
    L = queries.shape[2]
    if L == 1:
        if mask not in ("none", None):
            raise ValueError("decode (L == 1) takes no mask (BaseKVCache.makeMask returns .none)")
    else:
        if mask != "causal":
            raise ValueError("a multi-token pass takes the causal mask (BaseKVCache.makeMask(n > 1))")
        if window is not None or sinks is not None:
            raise ValueError("window and sinks are for a single token (L == 1)")
    if rope is not None:
        qw, kw, eps, offset = (tuple(norms) + (0.0,))[:4] if norms is not None else (None, None, 0.0, 0.0)
        queries, keys = cache.normRotate(queries, keys, qw, kw, eps, rope, weightOffset=offset)
    if L == 1 and not dense:
        return cache.appendDecode(keys, values, queries, scale)
    # nothing is appended that could not be attended to
    cache._check_q(queries, multi=L > 1)
    if keys.dim() != 4 or queries.shape[0] != keys.shape[0] or L != keys.shape[2]:
        raise ValueError("keys / values and queries disagree on B or L")
    if dense and L == 1:
        cache._check_sinks(sinks)
        cache._check_window(window)
        if queries.data_ptr() % 16:
            raise ValueError("queries must be 16-byte aligned")
    cache.append(keys, values)
    if L == 1:
        return cache.decodeDense(queries, scale, window=window, sinks=sinks)
    if L <= MAX_QUERIES and not dense:
        return cache.decodeMulti(queries, scale)
    return cache.prefill(queries, scale)


__all__ = ["attentionWithCacheUpdate"]
