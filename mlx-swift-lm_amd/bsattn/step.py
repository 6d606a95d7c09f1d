"""Step: requests that each bring their own number of new tokens, packed along
rows, as a tree of drafts or as a chain.

The general form of SpeculativeTokenIterator.speculateRound
(Libraries/MLXLMCommon/Evaluate.swift:841-931), which verifies one chain of
drafts per round and trims what was not accepted: map() says where the rows of
all requests lie in every layer's cache, attentionWithCacheUpdate(step=...)
appends them and attends to the trees, and BlockSparseKVCache.keep() keeps the
accepted paths.  Nothing in it waits for the host, and all of it can be
captured.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check, lib
from .cache import BlockSparseKVCache, _row_ids, _stream


class Step:
    """New tokens of up to 64 requests in `caches` (a model's layers, at the
    same lengths): `rows` rows in all, at most `maxTokens` of one request (at
    most 64 where they form trees).  Packed tensors are [rows, heads, D];
    request i's tokens are its rows starts[i] .. starts[i] + taken[i] - 1, and
    rows behind the last request's are nobody's.  One stream at a time; keep the
    object while calls or graphs that use it are pending.  A graph keeps the
    requests of its capture: once a captured step is mapped for others, its calls
    outside graphs are refused (another Step takes them).

    map() writes, on the device: starts [n + 1], taken [n] (0: the request does
    not fit), requests [rows] (-1: none), positions [rows] (what rotary
    positions take: cached tokens + depth in the tree), ancestors [rows] (bit a:
    the row sees its request's token a; None where maxTokens > 64), slots
    [caches, rows] (page * blockSize + place, -1: none) and ends [caches, n]
    (lengths with the new tokens)."""

    def __init__(self, caches: Sequence[BlockSparseKVCache], rows: int, maxTokens: int):
        caches = list(caches)
        if not 1 <= len(caches) <= _lib.STEP_CACHES:
            raise ValueError(f"a step takes 1 to {_lib.STEP_CACHES} caches (got {len(caches)})")
        if rows < 1 or maxTokens < 1:
            raise ValueError("rows and maxTokens must be at least 1")
        self.device, self._index = caches[0].device, caches[0]._index
        if any(c._index != self._index for c in caches):
            raise ValueError("the step's caches are on different GPUs")
        self.caches, self.rows, self.maxTokens = caches, int(rows), int(maxTokens)
        most = min(_lib.STEP_SEQS, min(c.desc.max_seqs for c in caches))

        def new(*shape, dtype=torch.int32):
            return torch.zeros(shape, dtype=dtype, device=self.device)
        self._starts, self._taken, self._ends = new(most + 1), new(most), new(len(caches) * most)
        self.requests, self.positions, self.slots = new(rows), new(rows), new(len(caches), rows)
        self.ancestors = new(rows, dtype=torch.int64) if maxTokens <= _lib.TREE_NODES else None
        # (the arrays are ready before any stream uses them)
        torch.cuda.current_stream(self.device).synchronize()
        self._most, self._n = most, 0
        self.starts, self.taken, self.ends = self._starts[:1], self._taken[:0], self._ends[:0].view(len(caches), 0)
        self._handles, self._held = (ctypes.c_void_p * len(caches))(), None
        self._c = _lib.Step(n_caches=len(caches), rows=self.rows, max_tokens=self.maxTokens, n_seqs=0,
                            starts=self._starts.data_ptr(), taken=self._taken.data_ptr(),
                            requests=self.requests.data_ptr(), positions=self.positions.data_ptr(),
                            ancestors=None if self.ancestors is None else self.ancestors.data_ptr(),
                            slots=self.slots.data_ptr(), ends=self._ends.data_ptr(), stamp=0)
        self._ref = ctypes.byref(self._c)

    def _check_ints(self, t: torch.Tensor, name: str, shape) -> int:
        if t.dtype is not torch.int32 or t.get_device() != self._index or not t.is_contiguous() or t.shape != shape:
            raise ValueError(f"{name} must be a contiguous int32 tensor {tuple(shape)} on {self.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def map(self, counts: torch.Tensor, parents: Optional[torch.Tensor] = None,
            seq_ids: Optional[Sequence[int]] = None) -> "Step":
        """counts [n] int32: tokens of each request (sequences seq_ids, default
        0 .. n - 1), whose pages are held already (reserve); parents [rows]
        int32: each node's parent among its request's tokens, -1 for one that
        follows the cached tokens (None: chains).  A request that brings more than
        maxTokens, or for which rows or pages do not suffice, is not taken."""
        n = counts.shape[0] if counts.dim() == 1 else 0
        if not 1 <= n <= self._most:
            raise ValueError(f"counts must hold 1 to {self._most} requests, got {tuple(counts.shape)}")
        at = self._check_ints(counts, "counts", (n,))
        up = None if parents is None else self._check_ints(parents, "parents", (self.rows,))
        held = [c._h for c in self.caches]
        if held != self._held:
            if None in held:
                raise ValueError("a cache of the step is closed")
            self._handles[:] = [h.value for h in held]
            self._held = held
        check(lib().bsattn_step_map(self._handles, self._ref, at, up, _row_ids(seq_ids, n), n, _stream(self.device)))
        if n != self._n:
            self._n = n
            self.starts, self.taken = self._starts[:n + 1], self._taken[:n]
            self.ends = self._ends[:len(self.caches) * n].view(len(self.caches), n)
        return self


__all__ = ["Step"]
