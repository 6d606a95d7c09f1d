"""Performance cases of a verification step over the paged cache: requests that
each bring their own number of new tokens, most of them a tree of drafts.

Four kinds of work, each one pass of run():

  map      from the requests' token counts (and the drafts' parents), all on the
           GPU: the packed rows' requests, positions, ancestors and page slots in
           every layer's cache;
  tree     attention of the drafted tokens over the paged cache: each sees what
           its request held before (or the last `window` positions of it) and
           its own ancestors;
  round    one round of a drafting server on one layer: map, append of the packed
           rows, tree attention, the accepted paths kept, attention of one token
           per request over what is then cached, and the drafts let go again;
  prompts  prompts of different lengths appended from one packed projection, then
           attention of their last tokens.

Packed tensors are views into a fused projection [rows, Hq + 2 Hkv, 128].
Queries, keys and values are N(0, 1).  Everything is made on the GPU from the
seed.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
SCALE = 1.0 / math.sqrt(D)


def _bsattn():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-swift-lm_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import bsattn
    return bsattn


# ---------------------------------------------------------------------------
# cases: P tokens are cached (spread over [P_min, P]), each request brings N new
# ones, or 1 to N of them (ragged)
# ---------------------------------------------------------------------------
def _case(name, kind, B, P, N, Hq=32, Hkv=8, Tb=64, dtype="bf16", bits=0, P_min=-1, ragged=False, chain=False,
          absent=False, window=0, sinks=False, layers=1):
    c = dict(kind=kind, B=B, P=P, P_min=P if P_min < 0 else P_min, N=N, Hq=Hq, Hkv=Hkv, Tb=Tb, dtype=dtype, bits=bits,
             ragged=ragged, chain=chain, absent=absent, window=window, sinks=sinks, layers=layers)
    return dict(c, name=name) if name else c


def _map(name, B, P, N, layers, **more):
    return _case(name, "map", B, P, N, Hq=1, Hkv=1, dtype="f16", bits=4, layers=layers, **more)


def listed():
    return [
        # one user's drafts in one layer: launch and latency
        _map("map_b1_16_1layer", 1, 2000, 16, 1),
        # a serving batch's drafts, for all layers of a model at once
        _map("map_b32_ragged48_36layers", 32, 4000, 48, 36, P_min=500, ragged=True),
        # one user, a short context, a small tree: launch and latency
        _case("tree_b1_4k_16_f16", "tree", 1, 4080, 16, dtype="f16"),
        # 8 users at 32k tokens, trees of 16: the benchmark's headline geometry
        _case("tree_b8_32k_16_bf16", "tree", 8, 32752, 16),
        # the same with the largest trees: as many products as bytes
        _case("tree_b8_32k_64_bf16", "tree", 8, 32704, 64),
        # long contexts in int4 caches, a tree of an odd size
        _case("tree_b4_131k_25_int4", "tree", 4, 131047, 25, dtype="f16", bits=4),
        # very long contexts in int8 caches, wide query groups, a short chain of drafts
        _case("tree_b4_262k_6_int8_g16", "tree", 4, 262138, 6, Hq=64, Hkv=4, Tb=32, dtype="f16", bits=8, chain=True),
        # a serving batch of ragged trees on a sliding-window layer with sinks
        _case("tree_b32_ragged_window_f16", "tree", 32, 65000, 48, dtype="f16", P_min=1000, ragged=True, window=4096,
              sinks=True),
        # one user's whole round
        _case("round_b1_8k_16_bf16", "round", 1, 8190, 16),
        # a batch's round over int8 caches, one token more than a tree of 32
        _case("round_b8_16k_33_int8", "round", 8, 16351, 33, dtype="f16", bits=8),
        # a serving batch's round, ragged lengths and trees
        _case("round_b32_ragged24_f16", "round", 32, 20000, 24, dtype="f16", P_min=300, ragged=True),
        # sixteen prompts of different lengths, packed
        _case("prompts_b16_ragged2048_bf16", "prompts", 16, 0, 2048, ragged=True, chain=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["map", "tree", "tree", "tree", "round", "round", "prompts"])
    if kind == "map":
        B, N, layers = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 48)
        P = _log(rng, 1, max(1, min(8000, 2000000 // (B * layers))))
        return _map(None, B, P, N, layers, P_min=rng.choice([P, 0]), Tb=rng.choice([32, 64]),
                    ragged=rng.random() < 0.5, chain=rng.random() < 0.4, absent=rng.random() < 0.2)
    Hkv, G = rng.choice([(8, 4), (8, 4), (4, 8), (4, 16), (8, 1), (2, 8), (16, 2)])
    bits = rng.choice([0, 0, 4, 8])
    common = dict(Hq=Hkv * G, Hkv=Hkv, Tb=rng.choice([32, 64, 64]), dtype="f16" if bits else rng.choice(["f16", "bf16"]),
                  bits=bits)
    token = Hkv * _token_bytes(common)
    if kind == "prompts":
        B, N = _log(rng, 1, 32), _log(rng, 1, 4096)
        N = max(1, min(N, int(1.2e8 / (Hkv * 2 * D * 2) / B)))
        P = rng.choice([0, _log(rng, 1, 4096)])
        return _case(None, kind, B, P, N, ragged=rng.random() < 0.7, chain=True, P_min=rng.choice([P, 0]), **common)
    B, N = _log(rng, 1, 32), _log(rng, 1, 64)
    P = _log(rng, 1, 262144)
    P = max(1, min(P, int((0.9e9 if kind == "tree" else 0.4e9) / token / B), int(2.2e11 / (4 * D * Hkv * G * N * B))))
    chain = rng.random() < 0.3
    return _case(None, kind, B, P, N, P_min=rng.choice([P, P, max(1, P // rng.randint(2, 8)), 1 if kind == "round" else 0]),
                 ragged=rng.random() < 0.5, chain=chain, absent=not chain and kind == "tree" and rng.random() < 0.3,
                 window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]) if kind == "tree" else 0,
                 sinks=kind == "tree" and rng.random() < 0.3, **common)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, *stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(random.Random(repr((seed,) + stream)).getrandbits(62))
    return g


def _normal(g, shape, dt):
    return torch.randn(shape, device="cuda", generator=g).to(dt)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(c):
    """Tokens that each request holds: P, or spread evenly over [P_min, P]."""
    return [c["P_min"] + int((c["P"] - c["P_min"]) * (((b + 1) * 0.6180339887498949) % 1.0)) for b in range(c["B"])]


def _counts(c):
    """New tokens of each request: N, or spread over [1, N], of prompts [N / 4, N]."""
    least = max(1, c["N"] // 4) if c["kind"] == "prompts" else 1
    return [least + int((c["N"] + 1 - least) * (((b + 1) * 0.7548776662466927) % 1.0)) if c["ragged"] else c["N"]
            for b in range(c["B"])]


def _parents(c, seed, counts):
    """Each request's nodes' parents: an earlier node, -1 for what follows the cached tokens, -2 where a place of the
    tree is not used."""
    r = random.Random(repr((seed, 1)))
    return [[-2 if c["absent"] and r.random() < 0.2 else r.randint(max(-1, j - 8), j - 1) if j else -1
             for j in range(n)] for n in counts]


def _paths(parents):
    """The nodes from the root to each node, itself included; [] where it is absent."""
    out = []
    for j, p in enumerate(parents):
        out.append([] if p < -1 or p >= j or (p >= 0 and not out[p]) else (out[p] if p >= 0 else []) + [j])
    return out


def _kept(c, seed, counts, parents):
    """An accepted path of each request, from nothing to the whole way to some node."""
    r = random.Random(repr((seed, 2)))
    out = []
    for n, p in zip(counts, parents):
        path = list(range(n)) if c["chain"] else r.choice(_paths(p))
        out.append(path[:r.randint(0, len(path))])
    return out


def _kv(c, seed, b, n):
    """Keys and values [Hkv, n, D] of the n tokens that request b holds."""
    g, dt = _gen(seed, 4, b), DTYPES[c["dtype"]]
    return _normal(g, (c["Hkv"], n, D), dt), _normal(g, (c["Hkv"], n, D), dt)


def _projected(c, seed, rows):
    """Queries, keys and values [rows, heads, D] of the new tokens: views into the fused projection."""
    x = _normal(_gen(seed, 5), (rows, c["Hq"] + 2 * c["Hkv"], D), DTYPES[c["dtype"]])
    return x[:, :c["Hq"]], x[:, c["Hq"]:c["Hq"] + c["Hkv"]], x[:, c["Hq"] + c["Hkv"]:]


def _last(c, seed):
    """One query per request."""
    return _normal(_gen(seed, 6), (c["B"], c["Hq"], 1, D), DTYPES[c["dtype"]])


def _sinks(c, seed):
    """A logit per query head, near the largest of a few thousand scores."""
    return torch.randn(c["Hq"], device="cuda", generator=_gen(seed, 7)) + 4.0


def _div(a, b):
    return (a.double() / b.double()).float()  # correctly rounded: a code at a border is everywhere the same


def _codes(x, bits):
    """Affine codes [..., D], scales and biases [..., D / 64] (fp16) of x, one of each per 64 dims."""
    x = x.float().reshape(*x.shape[:-1], D // 64, 64)
    mn, mx = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    bins = float((1 << bits) - 1)
    scale = torch.clamp(_div(mx - mn, torch.full_like(mn, bins)), min=1e-7)
    side = mn.abs() > mx.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, mn, mx)
    q0 = _div(edge, scale).round()
    scale = torch.where(q0 != 0, _div(edge, torch.where(q0 != 0, q0, torch.ones_like(q0))), scale)
    bias = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    codes = _div(x - bias, scale).round().clamp(0, bins)
    return codes.reshape(*codes.shape[:-2], D), scale[..., 0].half(), bias[..., 0].half()


def _words(codes, bits):
    """Codes [..., D] packed into 32-bit words, lowest first."""
    per = 32 // bits
    w = codes.to(torch.int64).reshape(*codes.shape[:-1], D // per, per)
    w = (w << (bits * torch.arange(per, device="cuda"))).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _stored(c, x):
    """What a cache holds of x: [x], or [words, scales, biases]."""
    if not c["bits"]:
        return [x]
    codes, scale, bias = _codes(x, c["bits"])
    return [_words(codes, c["bits"]), scale, bias]


def _inputs(c, seed):
    counts = _counts(c)
    parents = _parents(c, seed, counts)
    st = {"kind": c["kind"], "counts": _ints(counts), "rows": sum(counts),
          "parents": None if c["chain"] else _ints([p for t in parents for p in t])}
    if c["kind"] != "map":
        st["q"], st["k"], st["v"] = _projected(c, seed, sum(counts))
    if c["kind"] in ("round", "prompts"):
        st["last"] = _last(c, seed)
    if c["kind"] == "round":
        kept = _kept(c, seed, counts, parents)
        st["kept"] = _ints([k + [0] * (c["N"] - len(k)) for k in kept])
        st["n_kept"], st["none"] = _ints([len(k) for k in kept]), _ints([0] * c["B"])
    st["sinks"] = _sinks(c, seed) if c["sinks"] else None
    return st, counts


def _prepare_own(c, seed):
    """The layers' caches with the requests' tokens so far, pages reserved for the new ones, and the step."""
    bs = _bsattn()
    st, counts = _inputs(c, seed)
    held = _lengths(c)
    blocks = max(-(-(n + m) // c["Tb"]) for n, m in zip(held, counts))
    caches = [bs.BlockSparseKVCache(max_seqs=c["B"], num_q_heads=c["Hq"], num_kv_heads=c["Hkv"], head_dim=D,
                                    block_size=c["Tb"], dtype=DTYPES[c["dtype"]], kv_bits=c["bits"],
                                    max_blocks_per_seq=max(1, blocks), device=0) for _ in range(c["layers"])]
    for b, n in enumerate(held):
        if n:
            k, v = _kv(c, seed, b, n)
            k, v = (k[None], v[None]) if not c["bits"] else (_stored(c, k[None]), _stored(c, v[None]))
            for cache in caches:
                if c["bits"]:
                    cache.appendQuantized(tuple(k), tuple(v), seq_ids=[b])
                else:
                    cache.append(k, v, seq_ids=[b])
            del k, v
    for cache in caches:
        for b, m in enumerate(counts):
            cache.reserve(m, seq_ids=[b])
    step = bs.Step(caches, rows=st["rows"], maxTokens=c["N"])
    st.update(bs=bs, cache=caches[0], step=step, window=c["window"] or None)
    if c["kind"] in ("tree", "prompts"):
        step.map(st["counts"], st["parents"])
        if c["kind"] == "tree":
            caches[0].appendPacked(st["k"], st["v"], step)
    return st


def _tables(c, held, counts):
    """Each request's pages: those of what it holds, then those of what it brings, taken in order."""
    Tb, tables, at = c["Tb"], [], 0
    for n in held:
        tables.append(list(range(at, at + -(-n // Tb))))
        at += len(tables[-1])
    for t, n, m in zip(tables, held, counts):
        more = -(-(n + m) // Tb) - len(t)
        t.extend(range(at, at + more))
        at += more
    return tables, at


def _prepare_plain(c, seed):
    """Pools of pages [pages, Hkv, Tb, ...] with the requests' tokens so far, and their tables."""
    st, counts = _inputs(c, seed)
    held, Tb = _lengths(c), c["Tb"]
    tables, pages = _tables(c, held, counts)
    width = max(1, max(len(t) for t in tables))
    st.update(c=c, held=torch.tensor(held, device="cuda"), table=_ints([t + [0] * (width - len(t)) for t in tables]),
              pages_held=_ints([len(t) for t in tables]), most=max(n + m for n, m in zip(held, counts)))
    if c["kind"] == "map":
        return st
    shapes = [D] if not c["bits"] else [D * c["bits"] // 32, 2, 2]
    types = [DTYPES[c["dtype"]]] if not c["bits"] else [torch.int32, torch.float16, torch.float16]
    st["pools"] = [torch.zeros((max(1, pages), c["Hkv"], Tb, w), dtype=t, device="cuda") for w, t in zip(shapes, types)
                   for _ in (0, 1)]
    st["pools"] = st["pools"][0::2] + st["pools"][1::2]  # K's, then V's
    for b, n in enumerate(held):
        if n:
            parts = [t for x in _kv(c, seed, b, n) for t in _stored(c, x)]
            at, have = tables[b][0], -(-n // Tb)
            for pool, t in zip(st["pools"], parts):
                full = torch.zeros((c["Hkv"], have * Tb, t.shape[-1]), dtype=t.dtype, device="cuda")
                full[:, :n] = t
                pool[at:at + have] = full.reshape(c["Hkv"], have, Tb, -1).transpose(0, 1)
            del parts
    if c["kind"] in ("tree", "prompts"):
        st["step"] = _map_plain(st)
        if c["kind"] == "tree":
            _append_plain(st, st["step"])
    return st


def prepare(case, seed):
    """The requests' new tokens, and the caches (pages reserved) with what they hold."""
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_own(s):
    step, cache = s["step"], s["cache"]
    if s["kind"] == "map":
        step.map(s["counts"], s["parents"])
        return step.starts, step.taken, step.requests, step.positions, step.ancestors, step.slots, step.ends
    if s["kind"] == "tree":
        return cache.attendTree(s["q"], step, SCALE, window=s["window"], sinks=s["sinks"])
    if s["kind"] == "prompts":
        cache.appendPacked(s["k"], s["v"], step)
        return cache.decodeDense(s["last"], SCALE)
    step.map(s["counts"], s["parents"])
    out = s["bs"].attentionWithCacheUpdate(s["q"], s["k"], s["v"], cache, SCALE, step=step)
    cache.keep(step, s["kept"], s["n_kept"])
    after = cache.decodeDense(s["last"], SCALE)
    cache.keep(step, s["kept"], s["none"])
    return out, after


def _map_plain(s):
    c, n = s["c"], s["held"]
    counts, rows, width = s["counts"].long(), s["rows"], s["table"].shape[1]
    behind = torch.cumsum(counts, 0)
    starts = torch.cat([torch.zeros_like(behind[:1]), behind])
    fits = (counts <= c["N"]) & (behind <= rows) & (n + counts <= s["pages_held"] * c["Tb"])
    taken = torch.where(fits, counts, torch.zeros_like(counts))
    row = torch.arange(rows, device="cuda")
    req = torch.searchsorted(behind, row, right=True).clamp(max=c["B"] - 1)
    node = row - starts[req]
    there = node < taken[req]
    if s["parents"] is None:
        depth = node
        ancestors = (torch.ones_like(node) << (node + 1).clamp(max=63)) - 1
        ancestors = torch.where(node >= 63, torch.full_like(node, -1), ancestors)
    else:
        up = s["parents"].long()
        lost = (up < -1) | (up >= node)
        root = lost | (up < 0)
        at = torch.where(root, row, starts[req] + up)
        ancestors, depth = torch.ones_like(node) << node, torch.where(root, 0, 1)
        for _ in range(6):  # each time twice as far towards the root
            ancestors, lost = ancestors | ancestors[at], lost | lost[at]
            depth, at = depth + depth[at], at[at]
        ancestors, depth = torch.where(lost, 0, ancestors), torch.where(lost, 0, depth)
    pos = n[req] + node
    slots = s["table"][req, (pos // c["Tb"]).clamp(max=width - 1)].long() * c["Tb"] + pos % c["Tb"]
    zero = torch.zeros_like(node)
    return {"starts": starts.int(), "taken": taken.int(), "requests": torch.where(there, req, -1).int(),
            "positions": torch.where(there, n[req] + depth, zero).int(), "ancestors": torch.where(there, ancestors, zero),
            "slots": torch.where(there, slots, -1).int().expand(c["layers"], -1).contiguous(),
            "ends": (n + taken).int().expand(c["layers"], -1).contiguous()}


def _append_plain(s, m):
    """The new rows' keys and values into the pools, at their slots (all of them are taken)."""
    c, slot = s["c"], m["slots"][0].long()
    page, off = slot // c["Tb"], slot % c["Tb"]
    new = [t for x in (s["k"], s["v"]) for t in _stored(c, x)]
    for pool, t in zip(s["pools"], new):
        pool[page, :, off] = t


def _values_plain(c, parts):
    """Stored pages [B, n, Hkv, Tb, ...] -> [B * Hkv, n * Tb, D] in 32 bits."""
    if not c["bits"]:
        x = parts[0].float()
    else:
        w, scale, bias = parts
        shift = c["bits"] * torch.arange(32 // c["bits"], device="cuda", dtype=torch.int32)
        codes = ((w[..., None] >> shift) & ((1 << c["bits"]) - 1)).float().reshape(*w.shape[:-1], D // 64, 64)
        x = (codes * scale.float()[..., None] + bias.float()[..., None]).reshape(*w.shape[:-1], D)
    return x.transpose(1, 2).reshape(x.shape[0] * c["Hkv"], -1, D)


def _attend_plain(s, q, held, most, seen, depth, window):
    """q [B, N, Hq, D] of N nodes behind held [B] tokens (at most `most` with them), seen [B, N, N] of each other,
    at `depth` [B, N] -> [B, N, Hq, D] in 32 bits."""
    c, Tb = s["c"], s["c"]["Tb"]
    B, N = q.shape[:2]
    blocks = -(-most // Tb)
    first = torch.zeros_like(held)
    if window:
        first = (held - window + 1).clamp(min=0) // Tb
        blocks = min(blocks, (window + N + 2 * Tb) // Tb)
    at = (first[:, None] + torch.arange(blocks, device="cuda")).clamp(max=s["table"].shape[1] - 1)
    pages = torch.gather(s["table"].long(), 1, at)
    t = (first[:, None] * Tb + torch.arange(blocks * Tb, device="cuda"))[:, None]  # [B, 1, T] positions
    node = t - held[:, None, None]
    near = torch.ones_like(seen) if not window else depth[:, None, :] > depth[:, :, None] - window
    tree = torch.gather(seen & near, 2, node.clamp(0, N - 1).expand(-1, N, -1)) & (node >= 0) & (node < N)
    old = (node < 0) & torch.diagonal(seen, 0, 1, 2)[:, :, None]
    if window:
        old = old & (t > (held[:, None] + depth)[:, :, None] - window)
    mask = (tree | old)[:, None, :, None]  # [B, 1, N, 1, T]
    half = len(s["pools"]) // 2
    k, v = (_values_plain(c, [p[pages] for p in part]) for part in (s["pools"][:half], s["pools"][half:]))
    G = c["Hq"] // c["Hkv"]
    x = q.float().reshape(B, N, c["Hkv"], G, D).transpose(1, 2).reshape(B * c["Hkv"], N * G, D) * SCALE
    scores = torch.bmm(x, k.transpose(1, 2).contiguous()).reshape(B, c["Hkv"], N, G, -1)
    scores = torch.where(mask, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        top = torch.maximum(top, s["sinks"].reshape(1, c["Hkv"], 1, G, 1))
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].reshape(1, c["Hkv"], 1, G, 1) - top)
    out = torch.bmm(p.reshape(B * c["Hkv"], N * G, -1), v.contiguous()).reshape(B, c["Hkv"], N, G, D)
    return torch.where(total > 0, out / total, 0.0).transpose(1, 2).reshape(B, N, c["Hq"], D)


def _tree_plain(s, m):
    c = s["c"]
    N, taken = c["N"], m["taken"].long()
    node = torch.arange(N, device="cuda")
    row = (m["starts"][:-1].long()[:, None] + node).clamp(max=s["rows"] - 1)
    there = node < taken[:, None]
    ancestors = torch.where(there, m["ancestors"][row], 0)
    seen = ((ancestors[:, :, None] >> node) & 1).bool()
    depth = m["positions"][row].long() - s["held"][:, None]
    out = _attend_plain(s, s["q"][row], s["held"], s["most"], seen, depth, c["window"])
    return out[there].to(s["q"].dtype)


def _one_plain(s, length):
    """The last queries over the first length [B] tokens of each request."""
    one = torch.ones((s["c"]["B"], 1, 1), dtype=torch.bool, device="cuda")
    out = _attend_plain(s, s["last"].transpose(1, 2), length - 1, s["most"], one, torch.zeros_like(one[:, 0]).long(), 0)
    return out.transpose(1, 2).to(s["last"].dtype)


def _run_plain(s):
    if s["kind"] == "map":
        m = _map_plain(s)
        return m["starts"], m["taken"], m["requests"], m["positions"], m["ancestors"], m["slots"], m["ends"]
    if s["kind"] == "tree":
        return _tree_plain(s, s["step"])
    if s["kind"] == "prompts":
        _append_plain(s, s["step"])
        return _one_plain(s, s["held"] + s["step"]["taken"].long())
    m = _map_plain(s)
    _append_plain(s, m)
    out = _tree_plain(s, m)
    # the kept nodes move to the first of the new slots
    Tb, n = s["c"]["Tb"], torch.arange(s["c"]["N"], device="cuda")
    there = n < s["n_kept"].long()[:, None]
    row = m["starts"][:-1].long()[:, None]
    to, of = m["slots"][0][(row + n)[there]].long(), m["slots"][0][(row + s["kept"].long())[there]].long()
    for pool in s["pools"]:
        pool[to // Tb, :, to % Tb] = pool[of // Tb, :, of % Tb]
    return out, _one_plain(s, s["held"] + s["n_kept"].long())


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _token_bytes(c):
    """Bytes of one cached token's key and value in one kv head."""
    return 2 * D * 2 if c["bits"] == 0 else 2 * (D * c["bits"] // 8 + 8)


def work(case):
    c = case
    held = _lengths(c)
    counts = _counts(c)
    rows = sum(counts)
    if c["kind"] == "map":
        per_row = 4 + 4 + 8 + (0 if c["chain"] else 4) + c["layers"] * (4 + 4 / c["Tb"])
        return {"bytes": int(rows * per_row + c["B"] * (12 + c["layers"] * 12)), "flops": 0}
    tok = c["Hkv"] * _token_bytes(c)
    new = rows * 2 * c["Hkv"] * D * 2
    one = 2 * c["B"] * c["Hq"] * D * 2
    if c["kind"] == "prompts":
        return {"bytes": int(new + 2 * rows * tok + sum(held) * tok + one), "flops": int(4 * D * c["Hq"] * (sum(held) + rows))}
    past = [min(n, c["window"] or n) for n in held]
    seen = sum(past)
    by = (seen + rows) * tok + 2 * rows * c["Hq"] * D * 2
    flops = 4 * D * c["Hq"] * sum(m * (n + m / 2) for n, m in zip(past, counts))
    if c["kind"] == "round":  # the rows are stored, half of a path is moved, and all that is cached is read once more
        by += new + rows * tok + seen * tok + one
        flops += 4 * D * c["Hq"] * seen
    return {"bytes": int(by), "flops": int(flops)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_values(c, x):
    if not c["bits"]:
        return x.double()
    codes, scale, bias = (t.double() for t in _codes(x, c["bits"]))
    return codes * scale.repeat_interleave(64, -1) + bias.repeat_interleave(64, -1)


def _exact_rows(q, k, v, hide, sinks):
    """q [n, D] over k, v [T, D], less what hide [n, T] says, in 64 bits; sinks [n] or None."""
    s = torch.where(hide, -math.inf, q @ k.t() * SCALE)
    if sinks is not None:
        s = torch.cat([s, sinks[:, None]], 1)
    total = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(total == -math.inf, 0.0, torch.exp(s[:, :k.shape[0]] - torch.where(total == -math.inf, 0.0, total)))
    return p @ v


def exact(case, seed):
    c = case
    if c["kind"] == "map":
        return None
    st, counts = _inputs(c, seed)
    held, G = _lengths(c), c["Hq"] // c["Hkv"]
    parents = _parents(c, seed, counts)
    kept = _kept(c, seed, counts, parents) if c["kind"] == "round" else None
    sinks = None if st["sinks"] is None else st["sinks"].double()
    out = torch.zeros((st["rows"], c["Hq"], D), dtype=torch.float64, device="cuda")
    after = torch.zeros((c["B"], c["Hq"], 1, D), dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, m) in enumerate(zip(held, counts)):
        rows = slice(first, first + m)
        first += m
        k0, v0 = _kv(c, seed, b, n)
        paths = [list(range(j + 1)) for j in range(m)] if c["chain"] else _paths(parents[b])
        hide = None
        if c["kind"] != "prompts":
            depth = [len(p) - 1 for p in paths]
            hide = torch.ones((m, n + m), dtype=torch.bool)
            for j, path in enumerate(paths):
                if path:
                    lo = max(0, n + depth[j] - c["window"] + 1) if c["window"] else 0
                    hide[j, lo:n] = False
                    hide[j, [n + a for a in path if not c["window"] or depth[a] > depth[j] - c["window"]]] = False
            hide = hide.repeat_interleave(G, 0).cuda()
        for h in range(c["Hkv"]):
            heads = slice(h * G, (h + 1) * G)
            kn, vn = _exact_values(c, st["k"][rows, h]), _exact_values(c, st["v"][rows, h])
            kp, vp = _exact_values(c, k0[h]), _exact_values(c, v0[h])
            if c["kind"] != "prompts":
                q = st["q"][rows, heads].double().reshape(m * G, D)
                sk = None if sinks is None else sinks[heads].repeat(m)
                out[rows, heads] = _exact_rows(q, torch.cat([kp, kn]), torch.cat([vp, vn]), hide, sk).reshape(m, G, D)
            if c["kind"] != "tree":
                keep = kept[b] if kept is not None else list(range(m))
                ka, va = torch.cat([kp, kn[keep]]), torch.cat([vp, vn[keep]])
                see = torch.zeros((G, ka.shape[0]), dtype=torch.bool, device="cuda")
                after[b, heads, 0] = _exact_rows(st["last"][b, heads, 0].double(), ka, va, see, None)
    return after if c["kind"] == "prompts" else out if c["kind"] == "tree" else (out, after)
