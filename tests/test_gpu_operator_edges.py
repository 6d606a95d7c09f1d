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
