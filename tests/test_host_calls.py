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
    from bsattn import cache as module, rope
    fake = Library()
    monkeypatch.setattr(module, "lib", lambda: fake)
    for m in (module, rope):
        monkeypatch.setattr(m, "_stream", lambda device: 0)
    c = object.__new__(bsattn.BlockSparseKVCache)
    c.device, c.dtype, c._h, c._lib = torch.device("cpu"), torch.float16, None, fake
    c.desc = _lib.Desc(max_seqs=4, num_q_heads=HQ, num_kv_heads=HKV, head_dim=D, block_size=64, group_size=64)
    c._hq, c._hkv, c._dim, c.nselMax = HQ, HKV, D, 4
    c._index = -1  # (of a host tensor)
    c._plain = lambda t, shape: t.shape == shape and t.dtype is c.dtype and t.is_contiguous()
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


def _calls(cache, ids):
    """Every call whose rows name their sequences."""
    q, kv, rope = _rows(2, HQ), _rows(2, HKV), type("Rope", (), {"index": -1, "_ref": None})()
    idx = torch.zeros((2, HKV, 4), dtype=torch.int32)
    words, scales = (torch.zeros(s, dtype=t) for s, t in (((2, HKV, 1, D // 8), torch.int32), ((2, HKV, 1, 2), torch.float16)))
    import bsattn
    return {"append": lambda: cache.append(kv, kv, seq_ids=ids), "appendStep": lambda: cache.appendStep(kv, kv, seq_ids=ids),
            "appendQuantized": lambda: cache.appendQuantized((words, scales, scales), (words, scales, scales), seq_ids=ids),
            "selectBlocks": lambda: cache.selectBlocks(q, seq_ids=ids), "attend": lambda: cache.attend(q, idx, 0.1, seq_ids=ids),
            "decode": lambda: cache.decode(q, 0.1, seq_ids=ids),
            "decodeNoAlloc": lambda: cache.decodeNoAlloc(q, 0.1, torch.empty_like(q), seq_ids=ids),
            "appendDecode": lambda: cache.appendDecode(kv, kv, q, 0.1, seq_ids=ids),
            "decodeMulti": lambda: cache.decodeMulti(q, 0.1, seq_ids=ids), "prefill": lambda: cache.prefill(q, 0.1, seq_ids=ids),
            "decodeDense": lambda: cache.decodeDense(q, 0.1, seq_ids=ids),
            "normRotate": lambda: cache.normRotate(q, kv, None, None, 0.0, rope, seq_ids=ids),
            "applyRotaryPosition": lambda: bsattn.applyRotaryPosition(rope, q, cache, seq_ids=ids)}


@pytest.mark.parametrize("ids,ok", [([], False), ([1], False), ([1, 0, 2], False), ([1, 0], True), (None, True)])
def test_one_sequence_id_for_each_row(cache, ids, ok):
    """The library reads as many ids as a call has rows: a list that is shorter
    would be read past its end."""
    for name, call in _calls(cache, ids).items():
        cache.desc.kv_bits = 4 if name == "appendQuantized" else 0
        cache._lib.calls.clear()
        if ok:
            call()
            assert len(cache._lib.calls) == 1, name
        else:
            with pytest.raises(ValueError, match="sequence ids"):
                call()
            assert cache._lib.calls == [], name


def test_swift_calls_state_their_rows():
    """As the Python calls: every list of sequences says how many the call reads."""
    import os
    import re
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swift", "Sources", "MLXLMBlockSparse")
    calls = [c for f in sorted(os.listdir(at)) for c in re.findall(r"withSeqIds\(([^{]*)\) \{", open(os.path.join(at, f)).read())]
    assert len(calls) >= 14 and all(re.fullmatch(r"[^,]+, rows: .+", c) for c in calls), calls
    assert "precondition(ids.count == rows" in open(os.path.join(at, "Device.swift")).read()
