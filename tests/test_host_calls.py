"""What the Python calls check before the library sees anything: a cache over a
library that only notes its calls, with tensors in host memory."""
from __future__ import annotations

import pytest
import torch

HQ, HKV, D = 8, 2, 128


class Library:
    """Every function of the library: notes its name, and succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def cache(monkeypatch):
    import bsattn
    from bsattn import _lib
    from bsattn import cache as module
    fake = Library()
    monkeypatch.setattr(module, "lib", lambda: fake)
    monkeypatch.setattr(module, "_stream", lambda device: 0)
    c = object.__new__(bsattn.BlockSparseKVCache)
    c.device, c.dtype, c._h, c._lib = torch.device("cpu"), torch.float16, None, fake
    c.desc = _lib.Desc(max_seqs=4, num_q_heads=HQ, num_kv_heads=HKV, head_dim=D, block_size=64, group_size=64)
    c._hq, c._hkv, c._dim, c.nselMax = HQ, HKV, D, 4
    c._index = -1  # (of a host tensor)
    return c


def _rows(B, H, L=1):
    return torch.zeros((B, H, L, D), dtype=torch.float16)


def _odd(B, H, L=1):
    """A contiguous tensor that does not start at a multiple of 16 bytes."""
    return torch.zeros(B * H * L * D + 1, dtype=torch.float16)[1:].view(B, H, L, D)


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("L", [1, 3, 20])
@pytest.mark.parametrize("bad", ["odd", "type", "heads", "batch", "tokens", "strided"])
def test_nothing_is_appended_that_cannot_be_attended_to(cache, dense, L, bad):
    """attentionWithCacheUpdate refuses queries before it appends: the cache
    is not left with tokens that a second try would append again."""
    from bsattn import attentionWithCacheUpdate
    if bad == "odd" and not (dense and L == 1):
        pytest.skip("only the dense decode asks for aligned queries")
    if bad in ("tokens", "strided") and L == 1:
        pytest.skip("one token: the same queries")
    q = {"odd": _odd(2, HQ, L), "type": _rows(2, HQ, L).float(), "heads": _rows(2, HKV, L), "batch": _rows(1, HQ, L),
         "tokens": _rows(2, HQ, L + 1), "strided": _rows(2, L, HQ).transpose(1, 2)}[bad]
    with pytest.raises(ValueError):
        attentionWithCacheUpdate(q, _rows(2, HKV, L), _rows(2, HKV, L), cache, 0.1, "none" if L == 1 else "causal",
                                 dense=dense)
    assert cache._lib.calls == []


@pytest.mark.parametrize("L,dense,last", [(1, True, "bsattn_decode_dense"), (3, True, "bsattn_prefill"),
                                          (3, False, "bsattn_decode_multi"), (20, False, "bsattn_prefill")])
def test_calls_of_a_pass(cache, L, dense, last):
    from bsattn import attentionWithCacheUpdate
    attentionWithCacheUpdate(_rows(2, HQ, L), _rows(2, HKV, L), _rows(2, HKV, L), cache, 0.1,
                             "none" if L == 1 else "causal", dense=dense)
    assert cache._lib.calls == ["bsattn_append", last]
