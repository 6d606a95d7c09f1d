"""A Swift cache that is made from another one, or from a prompt-cache file,
says whether its layer attends to every token: the new cache's default would
switch such a layer to the block selection without an error."""
from __future__ import annotations

import os
import re

SOURCES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swift", "Sources", "MLXLMBlockSparse")
# These make a cache that has no layer's setting to keep.
FRESH = {"newBlockSparseCache"}


def _functions(text):
    """(name, body) of every func of a file."""
    for m in re.finditer(r"\bfunc (\w+)[^{]*\{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield m.group(1), text[m.end():i]


def test_caches_made_from_others_keep_the_flag():
    seen = {}
    for f in sorted(os.listdir(SOURCES)):
        for name, body in _functions(open(os.path.join(SOURCES, f)).read()):
            if re.search(r"BlockSparseKVCache\(|\.init\(adopting", body):
                seen[name] = bool(re.search(r"\.attendsDensely = attendsDensely", body))
    assert set(seen) >= FRESH | {"copy", "toQuantized", "registerPromptCacheClass"}
    assert all(kept for name, kept in seen.items() if name not in FRESH), seen


def test_the_prompt_cache_class_takes_the_flag():
    text = open(os.path.join(SOURCES, "PromptCache.swift")).read()
    head = re.search(r"func registerPromptCacheClass\(([^)]*)\)", text).group(1)
    assert "attendsDensely: Bool = false" in head
