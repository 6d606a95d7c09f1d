"""Performance cases of the operators around the paged cache: rotary positions,
norms of queries and keys with the rotation, dense decode attention and forks.

Four kinds of work, each one pass of run():

  rotary  positions of x [B, H, L, 128] rotated into the heads' leading dims;
  norm    queries and keys of a fused projection normalised per head, scaled
          and rotated in the same pass, in the layout that the cache takes;
  dense   attention of one new token per sequence over the whole paged cache
          (or its last `window` tokens), with a sink logit per head or without;
  fork    prompts branched into several continuations that share their pages,
          one new token appended to each, attention over all of it, and the
          branches dropped again.

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
EPS = 1e-6


def _bsattn():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-swift-lm_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import bsattn
    return bsattn


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rotary(name, kind, B, L, Hq=32, Hkv=8, dtype="bf16", rot=128, interleaved=False, scaling="none", base=10000.0,
            start=0, spread=0, projection=True, offset=0.0):
    c = dict(kind=kind, B=B, L=L, Hq=Hq, Hkv=Hkv, dtype=dtype, rot=rot, interleaved=interleaved, scaling=scaling,
             base=base, start=start, spread=spread, projection=projection, offset=offset)
    return dict(c, name=name) if name else c


def _dense(name, B, T, Hq=32, Hkv=8, Tb=64, dtype="bf16", bits=0, T_min=-1, window=0, sinks=False):
    c = dict(kind="dense", B=B, T=T, T_min=T if T_min < 0 else T_min, Hq=Hq, Hkv=Hkv, Tb=Tb, dtype=dtype, bits=bits,
             window=window, sinks=sinks)
    return dict(c, name=name) if name else c


def _fork(name, prompts, branches, T, Hq=32, Hkv=8, Tb=64, dtype="bf16", bits=0):
    c = dict(kind="fork", prompts=prompts, branches=branches, B=prompts * branches, T=T, Hq=Hq, Hkv=Hkv, Tb=Tb,
             dtype=dtype, bits=bits)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one user: launch and latency
        _rotary("rotary_b1_1tok_f16", "rotary", 1, 1, dtype="f16", start=4095),
        # prompt chunks of a batch whose model rotates half of each head, interleaved, stretched by yarn
        _rotary("rotary_b8_2048_half_bf16", "rotary", 8, 2048, rot=64, interleaved=True, scaling="yarn"),
        # a serving batch's decode step: 32 users, 8k to 64k tokens each
        _rotary("norm_b32_1tok_bf16", "norm", 32, 1, start=8192, spread=57344),
        # chunked prompt processing in 512-token steps, batched
        _rotary("norm_b8_chunk512_f16", "norm", 8, 512, dtype="f16", scaling="llama3", base=500000.0, start=32256),
        # a whole prompt of an odd length behind a very long context, wide query groups, part of each head
        _rotary("norm_b1_8191_g16_bf16", "norm", 1, 8191, Hq=64, Hkv=4, rot=96, scaling="longrope", start=253953,
                offset=1.0),
        # one user, a short context: launch and latency
        _dense("dense_b1_4k_f16", 1, 4096, dtype="f16"),
        # 8 users at 32k tokens: the dense layers of the benchmark's headline geometry
        _dense("dense_b8_32k_bf16", 8, 32768),
        # long contexts in int4 caches
        _dense("dense_b4_131k_int4", 4, 131072, dtype="f16", bits=4),
        # very long contexts in int8 caches, wide query groups
        _dense("dense_b4_262k_int8_g16", 4, 262144, Hq=64, Hkv=4, Tb=32, dtype="f16", bits=8),
        # a serving batch of ragged lengths on a sliding-window layer with sinks
        _dense("dense_b32_ragged_window_f16", 32, 65536, dtype="f16", T_min=1000, window=4096, sinks=True),
        # eight samples of one prompt of an odd length
        _fork("fork_8_of_8191_bf16", 1, 8, 8191),
        # beam search: four prompts, four beams each, int8 caches
        _fork("fork_4x4_of_16001_int8", 4, 4, 16001, dtype="f16", bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "norm", "dense", "dense", "dense", "fork"])
    Hkv, G = rng.choice([(8, 4), (8, 4), (4, 8), (4, 16), (8, 1), (2, 8), (16, 2)])
    heads = dict(Hq=Hkv * G, Hkv=Hkv)
    if kind in ("rotary", "norm"):
        L = rng.choice([1, _log(rng, 2, 8192)])
        B = max(1, min(_log(rng, 1, 32), 40 * 16384 // (L * Hkv * (G + 1))))
        return _rotary(None, kind, B, L, dtype=rng.choice(["f16", "bf16"]), rot=rng.choice([128, 128, 64, 32, 96, 20]),
                       interleaved=rng.random() < 0.4,
                       scaling=rng.choice(["none", "none", "linear", "llama3", "yarn", "longrope"]),
                       base=rng.choice([10000.0, 500000.0, 1000000.0]), start=rng.choice([0, _log(rng, 1, 1 << 20)]),
                       spread=rng.choice([0, _log(rng, 1, 65536)]), projection=rng.random() < 0.75,
                       offset=rng.choice([0.0, 0.0, 1.0]), **heads)
    bits = rng.choice([0, 0, 4, 8])
    common = dict(Tb=rng.choice([32, 64, 64]), dtype="f16" if bits else rng.choice(["f16", "bf16"]), bits=bits, **heads)
    per_token = Hkv * _token_bytes(common)
    if kind == "dense":
        B = _log(rng, 1, 32)
        T = max(1, min(_log(rng, 1, 262144), int(1.0e9 / per_token / B)))
        return _dense(None, B, T, T_min=rng.choice([T, T, max(1, T // rng.randint(2, 8)), 0 if T > 64 else T]),
                      window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), sinks=rng.random() < 0.3, **common)
    prompts, branches = _log(rng, 1, 8), _log(rng, 2, 16)
    prompts = min(prompts, 64 // branches)
    T = max(1, min(_log(rng, 1, 32768), int(0.5e9 / per_token / (prompts * branches))))
    return _fork(None, prompts, branches, T, **common)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, *stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(random.Random(repr((seed,) + stream)).getrandbits(62))
    return g


def _normal(g, shape, dt):
    return torch.randn(shape, device="cuda", generator=g).to(dt)


def _scaling_config(name, rot):
    """The rope_scaling entry of a model's configuration, and its max_position_embeddings."""
    return {
        "none": (None, 8192),
        "linear": ({"rope_type": "linear", "factor": 4.0}, 32768),
        "llama3": ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                    "original_max_position_embeddings": 8192}, 131072),
        "yarn": ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768, "beta_fast": 32.0,
                  "beta_slow": 1.0}, 131072),
        "longrope": ({"rope_type": "longrope", "original_max_position_embeddings": 4096,
                      "long_factor": [1.0 + 0.25 * i for i in range(rot // 2)]}, 131072),
    }[name]


def _projected(c, seed):
    """Queries [B, Hq, L, D] and keys [B, Hkv, L, D]: views into a fused projection's rows, or dense tensors."""
    g, dt, H = _gen(seed, 1), DTYPES[c["dtype"]], c["Hq"] + 2 * c["Hkv"]
    if c["projection"]:
        x = _normal(g, (c["B"], c["L"], H, D), dt).transpose(1, 2)
        return x[:, :c["Hq"]], x[:, c["Hq"]:c["Hq"] + c["Hkv"]]
    return _normal(g, (c["B"], c["Hq"], c["L"], D), dt), _normal(g, (c["B"], c["Hkv"], c["L"], D), dt)


def _weights(c, seed):
    g, dt = _gen(seed, 2), DTYPES[c["dtype"]]
    return [((1.0 - c["offset"]) + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dt) for _ in range(2)]


def _positions(c, seed):
    """int32 [B, L]: each sequence's tokens follow each other from its own start."""
    r = random.Random(repr((seed, 3)))
    first = [c["start"] + r.randint(0, c["spread"]) for _ in range(c["B"])]
    return (torch.tensor(first, device="cuda")[:, None] + torch.arange(c["L"], device="cuda")[None]).to(torch.int32)


def _lengths(c):
    """Tokens of each sequence: T, or spread evenly over [T_min, T]."""
    if c["kind"] == "fork":
        return [c["T"]] * c["prompts"]
    return [c["T_min"] + int((c["T"] - c["T_min"]) * (((b + 1) * 0.6180339887498949) % 1.0)) for b in range(c["B"])]


def _kv(c, seed, b, n):
    """Keys and values [Hkv, n, D] of the n tokens that sequence b holds."""
    g, dt = _gen(seed, 4, b), DTYPES[c["dtype"]]
    return _normal(g, (c["Hkv"], n, D), dt), _normal(g, (c["Hkv"], n, D), dt)


def _new(c, seed):
    """Queries, keys and values of one new token per row."""
    g, dt = _gen(seed, 5), DTYPES[c["dtype"]]
    return (_normal(g, (c["B"], c["Hq"], 1, D), dt), _normal(g, (c["B"], c["Hkv"], 1, D), dt),
            _normal(g, (c["B"], c["Hkv"], 1, D), dt))


def _sinks(c, seed):
    """A logit per query head, near the largest of a few thousand scores."""
    return torch.randn(c["Hq"], device="cuda", generator=_gen(seed, 6)) + 4.0


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


def _cache(c, rows, tokens):
    bs = _bsattn()
    return bs.BlockSparseKVCache(max_seqs=rows, num_q_heads=c["Hq"], num_kv_heads=c["Hkv"], head_dim=D,
                                 block_size=c.get("Tb", 64), dtype=DTYPES[c["dtype"]], kv_bits=c.get("bits", 0),
                                 max_blocks_per_seq=max(1, -(-tokens // c.get("Tb", 64))), device=0)


def _prepare_own(c, seed):
    bs = _bsattn()
    if c["kind"] in ("rotary", "norm"):
        config, longest = _scaling_config(c["scaling"], c["rot"])
        rope = bs.initializeRope(c["rot"], c["base"], c["interleaved"], config, longest, device=0)
        q, k = _projected(c, seed)
        st = {"bs": bs, "kind": c["kind"], "rope": rope, "cache": _cache(c, c["B"], 64), "q": q,
              "pos": _positions(c, seed)}
        if c["kind"] == "norm":
            st.update(k=k, w=_weights(c, seed), offset=c["offset"])
        return st
    fork = c["kind"] == "fork"
    held = _lengths(c)
    # branches are the cache's first rows, the prompts the rows behind them
    first = c["B"] if fork else 0
    cache = _cache(c, first + len(held), c["T"] + (1 if fork else 0))
    cache.shuffleFreePages(seed)
    for b, n in enumerate(held):
        if n:
            k, v = _kv(c, seed, b, n)
            if c["bits"]:
                k, v = _stored(c, k[None]), _stored(c, v[None])
                cache.appendQuantized(tuple(k), tuple(v), seq_ids=[first + b])
            else:
                cache.append(k[None], v[None], seq_ids=[first + b])
            del k, v
    q, k, v = _new(c, seed)
    st = {"bs": bs, "kind": c["kind"], "cache": cache, "q": q}
    if fork:
        st.update(k=k, v=v, dst=list(range(c["B"])), src=[first + i // c["branches"] for i in range(c["B"])])
    else:
        st.update(window=c["window"] or None, sinks=_sinks(c, seed) if c["sinks"] else None)
    return st


def _prepare_plain(c, seed):
    if c["kind"] in ("rotary", "norm"):
        q, k = _projected(c, seed)
        theta, m = _frequencies(c)
        st = {"c": c, "q": q, "pos": _positions(c, seed), "theta": theta, "m": m}
        if c["kind"] == "norm":
            st.update(k=k, w=_weights(c, seed))
        return st
    # pools of pages [pages, Hkv, Tb, ...] in shuffled order, and each row's table
    held, Tb, fork = _lengths(c), c["Tb"], c["kind"] == "fork"
    need = [-(-n // Tb) for n in held]
    spare = 2 * c["B"] if fork else 0
    order = list(range(sum(need) + spare))
    random.Random(repr((seed, 7))).shuffle(order)
    pools, tables, at = None, [], 0
    for b, n in enumerate(held):
        pages = order[at:at + need[b]]
        at += need[b]
        tables.append(pages)
        if not n:
            continue
        parts = [t for x in _kv(c, seed, b, n) for t in _stored(c, x)]  # [Hkv, n, ...]
        if pools is None:
            pools = [torch.zeros((max(1, len(order)), c["Hkv"], Tb, t.shape[-1]), dtype=t.dtype, device="cuda")
                     for t in parts]
        at_pages = torch.tensor(pages, device="cuda")
        for pool, t in zip(pools, parts):
            full = torch.zeros((c["Hkv"], need[b] * Tb, t.shape[-1]), dtype=t.dtype, device="cuda")
            full[:, :n] = t
            pool[at_pages] = full.reshape(c["Hkv"], need[b], Tb, -1).transpose(0, 1)
        del parts
    q, k, v = _new(c, seed)
    return {"c": c, "pools": pools, "tables": tables, "held": held, "spare": order[at:], "q": q, "k": k, "v": v,
            "sinks": _sinks(c, seed) if c.get("sinks") else None}


def prepare(case, seed):
    """The projections, the rotation and its positions, or the caches with their conversations so far."""
    return _prepare_own(case, seed) if own else _prepare_plain(case, seed)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_own(s):
    bs, cache = s["bs"], s["cache"]
    if s["kind"] == "rotary":
        return bs.applyRotaryPosition(s["rope"], s["q"], cache, positions=s["pos"])
    if s["kind"] == "norm":
        return cache.normRotate(s["q"], s["k"], s["w"][0], s["w"][1], EPS, s["rope"], positions=s["pos"],
                                weightOffset=s["offset"])
    if s["kind"] == "dense":
        return cache.decodeDense(s["q"], SCALE, window=s["window"], sinks=s["sinks"])
    cache.fork(s["src"], s["dst"])
    out = bs.attentionWithCacheUpdate(s["q"], s["k"], s["v"], cache, SCALE, dense=True)
    cache.reset(s["dst"])
    return out


def _frequencies(c):
    """Radians per position of each pair, in 64 bits, and the factor on the rotated dims."""
    R, base, name = c["rot"], c["base"], c["scaling"]
    config, longest = _scaling_config(name, R)
    theta, m = [base ** (-2.0 * i / R) for i in range(R // 2)], 1.0
    if name == "linear":
        theta = [t / config["factor"] for t in theta]
    elif name == "llama3":
        f, lo, hi = config["factor"], config["low_freq_factor"], config["high_freq_factor"]
        first = config["original_max_position_embeddings"]
        for i, t in enumerate(theta):
            turns = first * t / (2.0 * math.pi)
            mix = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            theta[i] = mix * t + (1.0 - mix) * t / f
    elif name == "yarn":
        f, first = config["factor"], config["original_max_position_embeddings"]

        def pair(turns):
            return R * math.log(first / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        lo = max(math.floor(pair(config["beta_fast"])), 0)
        hi = min(math.ceil(pair(config["beta_slow"])), R - 1)
        for i, t in enumerate(theta):
            ramp = min(1.0, max(0.0, (i - lo) / (hi - lo if hi != lo else 0.001)))
            theta[i] = t * (1.0 - ramp) + t / f * ramp
        m = 0.1 * math.log(f) + 1.0
    elif name == "longrope":
        first = config["original_max_position_embeddings"]
        theta = [t / f for t, f in zip(theta, config["long_factor"])]
        m = math.sqrt(1.0 + math.log(longest / first) / math.log(first))
    return torch.tensor(theta, dtype=torch.float64, device="cuda"), m


def _rotate_plain(s, x):
    """x [B, H, L, D] in 32 bits -> the rotated heads in 32 bits."""
    c = s["c"]
    R = c["rot"]
    phi = s["pos"].double()[:, None, :, None] * s["theta"]
    cos, sin = (torch.cos(phi) * s["m"]).float(), (torch.sin(phi) * s["m"]).float()
    out = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = a * cos - b * sin, a * sin + b * cos
    return out


def _values_plain(c, parts):
    """Stored pages [n, Hkv, Tb, ...] -> [Hkv, n * Tb, D] in 32 bits."""
    if not c["bits"]:
        x = parts[0].float()
    else:
        w, scale, bias = parts
        shift = c["bits"] * torch.arange(32 // c["bits"], device="cuda", dtype=torch.int32)
        codes = ((w[..., None] >> shift) & ((1 << c["bits"]) - 1)).float().reshape(*w.shape[:-1], D // 64, 64)
        x = (codes * scale.float()[..., None] + bias.float()[..., None]).reshape(*w.shape[:-1], D)
    return x.transpose(0, 1).reshape(c["Hkv"], -1, D)


def _attend_plain(s, q, table, T, window, sinks):
    """q [Hq, D] of one row over the last `window` (0: all) of its T tokens."""
    c = s["c"]
    if T == 0:
        return torch.zeros_like(q)
    t0 = max(0, T - window) if window else 0
    j0 = t0 // c["Tb"]
    pages = torch.tensor(table[j0:-(-T // c["Tb"])], device="cuda")
    parts = [p[pages] for p in s["pools"]]
    half = len(parts) // 2
    k, v = (_values_plain(c, p)[:, t0 - j0 * c["Tb"]:T - j0 * c["Tb"]] for p in (parts[:half], parts[half:]))
    scores = torch.bmm(q.float().reshape(c["Hkv"], -1, D) * SCALE, k.transpose(1, 2).contiguous())
    top = scores.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks.reshape(c["Hkv"], -1, 1))
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks.reshape(c["Hkv"], -1, 1) - top)
    return (torch.bmm(p, v.contiguous()) / total).reshape(c["Hq"], D).to(q.dtype)


def _run_plain(s):
    c = s["c"]
    if c["kind"] == "rotary":
        return _rotate_plain(s, s["q"].float()).to(s["q"].dtype)
    if c["kind"] == "norm":
        out = []
        for x, w in zip((s["q"], s["k"]), s["w"]):
            f = x.float()
            f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * (w.float() + c["offset"])
            out.append(_rotate_plain(s, f).to(x.dtype))
        return tuple(out)
    q = s["q"][:, :, 0]
    if c["kind"] == "dense":
        rows = [_attend_plain(s, q[b], s["tables"][b], s["held"][b], c["window"], s["sinks"]) for b in range(c["B"])]
        return torch.stack(rows)[:, :, None]
    # every branch shares the prompt's full pages, and takes a page of its own for what follows them
    T, Tb, rows = c["T"], c["Tb"], []
    new = [t for x in (s["k"], s["v"]) for t in _stored(c, x[:, :, 0])]  # [B, Hkv, ...]
    for i in range(c["B"]):
        table = s["tables"][i // c["branches"]]
        page = s["spare"][i]
        branch = table[:T // Tb] + [page]
        for pool, x in zip(s["pools"], new):
            if T % Tb:
                pool[page] = pool[table[-1]]
            pool[page, :, T % Tb] = x[i]
        rows.append(_attend_plain(s, q[i], branch, T + 1, 0, None))
    return torch.stack(rows)[:, :, None]


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
    if c["kind"] in ("rotary", "norm"):
        rows = c["B"] * c["L"] * (c["Hq"] + (c["Hkv"] if c["kind"] == "norm" else 0))
        flops = rows * (3 * c["rot"] + (4 * D if c["kind"] == "norm" else 0))
        return {"bytes": rows * D * 2 * 2 + c["B"] * c["L"] * 4, "flops": flops}
    tok = c["Hkv"] * _token_bytes(c)
    io = 2 * c["B"] * c["Hq"] * D * 2
    if c["kind"] == "dense":
        seen = sum(min(n, c["window"] or n) for n in _lengths(c))
        return {"bytes": seen * tok + io, "flops": 4 * D * c["Hq"] * seen}
    # the prompts once, each branch's own copy of the last page's tokens, its new token read, stored and read
    tail = c["T"] % c["Tb"]
    by = c["prompts"] * c["T"] * tok + c["B"] * (tail * tok + 2 * c["Hkv"] * D * 2 + tok) + io
    return {"bytes": by, "flops": 4 * D * c["Hq"] * c["B"] * (c["T"] + 1)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_angles(c, seed):
    """Angles [B, 1, L, rot / 2] and the factor on the rotated dims."""
    R = c["rot"]
    config, longest = _scaling_config(c["scaling"], R)
    i = torch.arange(R // 2, dtype=torch.float64, device="cuda")
    wave = 2 * math.pi * torch.exp(2 * i / R * math.log(c["base"]))  # positions per turn
    m = 1.0
    if c["scaling"] == "linear":
        wave = wave * config["factor"]
    elif c["scaling"] == "llama3":
        n, lo, hi = config["original_max_position_embeddings"], config["low_freq_factor"], config["high_freq_factor"]
        keep = torch.clamp((n / wave - lo) / (hi - lo), 0, 1)
        wave = 1 / (keep / wave + (1 - keep) / (config["factor"] * wave))
    elif c["scaling"] == "yarn":
        n = config["original_max_position_embeddings"]
        edges = [R / 2 * math.log(n / (2 * math.pi * r), c["base"]) for r in (config["beta_fast"], config["beta_slow"])]
        lo, hi = max(0, math.floor(edges[0])), min(R - 1, math.ceil(edges[1]))
        stretch = torch.clamp((i - lo) / max(hi - lo, 0.001), 0, 1)
        wave = 1 / ((1 - stretch) / wave + stretch / (config["factor"] * wave))
        m = 1 + math.log(config["factor"]) / 10
    elif c["scaling"] == "longrope":
        n = config["original_max_position_embeddings"]
        wave = wave * torch.tensor(config["long_factor"], dtype=torch.float64, device="cuda")
        m = math.sqrt(1 + math.log(longest / n, n))
    return _positions(c, seed).double()[:, None, :, None] * (2 * math.pi / wave), m


def _exact_rotated(c, x, phi, m):
    """x [B, H, L, D] in 64 bits: each pair a complex number turned by phi."""
    R = c["rot"]
    turn = torch.polar(torch.full_like(phi, m), phi)
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2).contiguous())
        head = torch.view_as_real(z * turn).reshape(*x.shape[:-1], R)
    else:
        z = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., R:]], -1)


def _exact_row(q, k, v, sinks):
    """q [G, D] over k, v [T, D], in 64 bits; sinks [G] or None."""
    s = q @ k.t() * SCALE
    total = torch.logsumexp(s, -1) if sinks is None else torch.logsumexp(torch.cat([s, sinks[:, None]], 1), -1)
    return torch.exp(s - total[:, None]) @ v


def _exact_values(c, x):
    if not c["bits"]:
        return x.double()
    codes, scale, bias = (t.double() for t in _codes(x, c["bits"]))
    return codes * scale.repeat_interleave(64, -1) + bias.repeat_interleave(64, -1)


def exact(case, seed):
    c = case
    if c["kind"] in ("rotary", "norm"):
        phi, m = _exact_angles(c, seed)
        q, k = (x.double() for x in _projected(c, seed))
        if c["kind"] == "rotary":
            return _exact_rotated(c, q, phi, m)
        out = []
        for x, w in zip((q, k), _weights(c, seed)):
            norm = torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + EPS)
            out.append(_exact_rotated(c, x / norm * (w.double() + c["offset"]), phi, m))
        return tuple(out)
    fork = c["kind"] == "fork"
    G, held = c["Hq"] // c["Hkv"], _lengths(c)
    q, nk, nv = _new(c, seed)
    sinks = _sinks(c, seed).double() if c.get("sinks") else None
    out = torch.zeros((c["B"], c["Hq"], 1, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(held):
        if not n:
            continue
        t0 = 0 if fork or not c["window"] else max(0, n - c["window"])
        k, v = (x[:, t0:] for x in _kv(c, seed, b, n))
        for h in range(c["Hkv"]):
            heads = slice(h * G, (h + 1) * G)
            kk, vv = _exact_values(c, k[h]), _exact_values(c, v[h])
            for i in range(b * c["branches"], (b + 1) * c["branches"]) if fork else (b,):
                ki, vi = kk, vv
                if fork:
                    ki, vi = torch.cat([kk, _exact_values(c, nk[i, h])]), torch.cat([vv, _exact_values(c, nv[i, h])])
                out[i, heads, 0] = _exact_row(q[i, heads, 0].double(), ki, vi, None if sinks is None else sinks[heads])
    return out
