"""Operators around a key / value cache held in 8 bits, and around one that is kept short, on one MI355X: norms of queries
and keys per head with the rotary embedding and the append in one pass, attention over the 8-bit cache, the attention
weight that every cached position gathers, and the eviction of the positions that gathered least.

An 8-bit cache holds e4m3 numbers c (OCP form) and, per block of consecutive positions and head, one scale s, a power of
two: value = s * c.  A block's first token sets s = 2^(floor(log2(largest magnitude)) - 5); s stays until a later token
passes 448 s, when it is set anew from that token and what the block holds is rounded to the new scale.
`own` False computes the plain form in elementary torch operations from the same buffers; True calls saga_amd.

Head layouts and widths are those of the decoder shapes in saga_amd/decoder.py (12 query / 1 key / 2 value heads of
128, and 15 / 1 / 5 of 64, each also with as many key heads as value heads); lengths, batches and positions are those
of bench.py and of the latency grid of saga_amd/speedup.py (batch 1-32, 4k-64k positions).
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn
EPS = 1e-6
# query, key and value heads, head dim
HEADS = {"12/1/2x128": (12, 1, 2, 128), "12/2/2x128": (12, 2, 2, 128), "15/1/5x64": (15, 1, 5, 64),
         "15/5/5x64": (15, 5, 5, 64)}


def listed():
    return [
        # One token of the smallest model into a 16-bit cache: the least work of a decode step, a launch's latency.
        {"name": "norm_b1", "kind": "norm", "heads": "15/1/5x64", "b": 1, "n": 0, "L": 4096, "dtype": "bf16"},
        # A prompt's tokens into one row of a 16-bit cache.
        {"name": "norm_prompt_4001", "kind": "norm", "heads": "12/1/2x128", "b": 2, "n": 4001, "L": 4352, "dtype": "bf16"},
        # A decode step's new tokens into an 8-bit cache, each somewhere in a block, and their rows read back.
        {"name": "norm8_b8", "kind": "norm8", "heads": "12/1/2x128", "b": 8, "n": 0, "L": 33024, "block": 64,
         "dtype": "bf16"},
        # Four prompts of different lengths behind what their rows hold, read back for their attention.
        {"name": "norm8_ragged_4", "kind": "norm8", "heads": "15/5/5x64", "b": 4, "n": 9001, "L": 8195, "block": 32,
         "dtype": "f16"},
        # One sequence of the small model over a short cache: latency.
        {"name": "dense8_b1_4k", "kind": "dense8", "heads": "15/1/5x64", "b": 1, "L": 4096, "fill": 4096, "block": 32,
         "dtype": "bf16", "mask": False, "trace": False},
        # A served batch of different lengths with left padding masked off, plain GQA, f16.
        {"name": "dense8_b4_8k_ragged", "kind": "dense8", "heads": "15/5/5x64", "b": 4, "L": 8195, "fill": 0, "block": 128,
         "dtype": "f16", "mask": True, "trace": False},
        # The headline decode's attention: static cache, 32769 filled positions.
        {"name": "dense8_b8_32k", "kind": "dense8", "heads": "12/1/2x128", "b": 8, "L": 33024, "fill": 32769, "block": 64,
         "dtype": "bf16", "mask": False, "trace": False},
        # The largest cell of the latency grid, every position's weight gathered too.
        {"name": "dense8_b32_64k_trace", "kind": "dense8", "heads": "12/1/2x128", "b": 32, "L": 65544, "fill": 65541,
         "block": 64, "dtype": "bf16", "mask": False, "trace": True},
        # The same weights over a 16-bit cache, whose attention selects or is dense: one short sequence, latency.
        {"name": "trace_b1_4k", "kind": "trace", "heads": "15/5/5x64", "b": 1, "L": 4099, "fill": 4097, "dtype": "f16",
         "mask": False},
        # The headline decode's.
        {"name": "trace_b8_32k", "kind": "trace", "heads": "12/1/2x128", "b": 8, "L": 33024, "fill": 32769, "dtype": "bf16",
         "mask": False},
        # The headline cache, 16 bits, cut to its half.
        {"name": "evict_b8_32k", "kind": "evict", "heads": "12/1/2x128", "b": 8, "L": 33024, "fill": 32769, "keep": 16384,
         "recent": 1024, "dtype": "bf16"},
        # A served batch of different lengths in 8 bits cut to an odd length (some rows are shorter), read back.
        {"name": "evict8_b4_8k_ragged", "kind": "evict8", "heads": "15/5/5x64", "b": 4, "L": 8195, "fill": 0, "keep": 3001,
         "recent": 333, "block": 32, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm8", "norm8", "dense8", "dense8", "dense8", "trace", "evict", "evict8"])
    c = {"kind": kind, "heads": rng.choice(list(HEADS)), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind.endswith("8"):
        c["block"] = rng.choice([32, 64, 128])
    c["b"] = _log(rng, 1, 32)
    if kind.startswith("norm"):
        c["n"] = rng.choice([0, _log(rng, 2, 9000)])
        if c["n"]:
            c["b"] = min(c["b"], 8)
        c["L"] = c["n"] + _log(rng, 100, 4000)
        return c
    c["L"] = _log(rng, 100, min(65000, (250000 if c["kind"].startswith("evict") else 600000) // c["b"]))
    c["fill"] = rng.choice([0, c["L"], max(1, c["L"] - c["L"] // 50)])
    if kind.startswith("evict"):
        c["keep"] = rng.randint(1, max(1, c["L"] * 3 // 4))
        c["recent"] = rng.choice([0, rng.randint(0, c["keep"]), c["keep"] // 8])
        return c
    c["mask"] = rng.random() < 0.25
    if kind == "dense8":
        c["trace"] = rng.random() < 0.4
    return c


# ------------------------------------------------------------------- the 8-bit form

def _pow2(e, dtype):
    """2^e of whole e >= -126."""
    return ((e.int() + 127) << 23).view(torch.float32).to(dtype)


def _scale(top):
    """The scale that a block's largest magnitude asks for (0 where that is 0)."""
    m, e = torch.frexp(top)      # top = m 2^e, m in [1/2, 1)
    return torch.where(top > 0, _pow2((e - 6).clamp(min=-100), top.dtype), torch.zeros_like(top))


def _e4m3(x):
    """x rounded to the nearest e4m3 number, ties to even, in x's own precision (|x| at most 448)."""
    m, e = torch.frexp(x)
    step = _pow2((e - 1).clamp(min=-6) - 3, x.dtype)
    return torch.round(x / step) * step


def _codes(x):
    """Bytes of the e4m3 numbers x."""
    return x.float().to(F8).view(torch.uint8)


def _open(codes, dtype=torch.float32):
    return codes.view(F8).to(dtype)


def _over(x, s):
    return x / torch.where(s > 0, s, torch.ones_like(s))


def _quantise(x, block):
    """Codes and scales [..., ceil(L / block)] of x [..., L, d], a block at a time."""
    L, d = x.shape[-2:]
    nb = -(-L // block)
    g = torch.nn.functional.pad(x, (0, 0, 0, nb * block - L)).unflatten(-2, (nb, block))
    s = _scale(g.abs().amax((-1, -2)))
    c = _e4m3(_over(g, s[..., None, None])).flatten(-3, -2)[..., :L, :]
    return _codes(c), s


def _values(codes, s, block, dtype=torch.float32):
    """s * c of codes [..., L, d] and scales [..., blocks]."""
    return _open(codes, dtype) * s.to(dtype).repeat_interleave(block, -1)[..., : codes.shape[-2], None]


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device=DEV, dtype=dtype)


def _lens(c):
    L, b = c["L"], c["b"]
    return [c["fill"]] * b if c["fill"] else [L - (3 * L // 4) * i // b for i in range(b)]


def _prompt_lens(c):
    """Tokens of the rows of a ragged append: about n in all, the first rows the longest."""
    b, n = c["b"], c["n"]
    return [max(n * 2 * (b - i) // (b * (b + 1)), 1 if i == 0 else 0) for i in range(b)]


def _cache8(g, c, lens):
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    b, L, block = c["b"], c["L"], c["block"]
    nb = -(-L // block)
    cache = {}
    outlier = 1 + 3 * (torch.rand(d, generator=g, device=DEV) < 0.05)   # keys have a few long dims
    for h, name, by in ((k_h, "k", outlier), (v_h, "v", 1)):
        cache[name + "_codes"] = torch.zeros(b, h, L, d, dtype=torch.uint8, device=DEV)
        cache[name + "_scales"] = torch.zeros(b, h, nb, device=DEV)
        for i in range(b):
            if lens[i]:
                codes, s = _quantise(_randn(g, h, lens[i], d) * by, block)
                cache[name + "_codes"][i, :, : lens[i]] = codes
                cache[name + "_scales"][i, :, : s.shape[-1]] = s
    return cache


def _empty8(c, L):
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    nb = -(-L // c["block"])
    return {f"{name}_{part}": t for h, name in ((k_h, "k"), (v_h, "v"))
            for part, t in (("codes", torch.zeros(c["b"], h, L, d, dtype=torch.uint8, device=DEV)),
                            ("scales", torch.zeros(c["b"], h, nb, device=DEV)))}


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c, g = case, _gen(seed)
    st = {"case": c}
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    b, L, dt = c["b"], c["L"], DTYPES[c["dtype"]]
    if c["kind"] in ("norm", "norm8"):
        st["q_norm"], st["k_norm"] = ((1 + 0.2 * _randn(g, d)).to(dt) for _ in range(2))
        if c["kind"] == "norm":
            n = c["n"] or b
            st["k"], st["v"] = (torch.zeros(b, h, L, d, dtype=dt, device=DEV) for h in (k_h, v_h))
            if c["n"]:   # a prompt into batch row b - 1, behind whatever of it is there
                st["pos"], st["batch"] = torch.arange(n, dtype=torch.int32, device=DEV) + (L - n) // 2, _int32([b - 1] * n)
            else:        # one token of every batch row
                st["pos"] = torch.randint(L // 2, L, (n,), generator=g, device=DEV, dtype=torch.int32)
                st["batch"] = None
        else:
            lens = _prompt_lens(c) if c["n"] else [1] * b
            n = sum(lens)
            start = [int(x * (L - k)) for x, k in zip(torch.rand(b, generator=torch.Generator().manual_seed(seed)).tolist(), lens)]
            st["cache"] = _cache8(g, c, start)
            st["start"] = _int32(start)
            st["offsets"] = _int32([sum(lens[:i]) for i in range(b + 1)]) if c["n"] else None
            st["batch"] = _int32([i for i in range(b) for _ in range(lens[i])])
            st["pos"] = _int32([start[i] + j for i in range(b) for j in range(lens[i])])
        st["qkv"] = _randn(g, n, (q_h + k_h + v_h) * d).to(dt)
        i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
        a = st["pos"].double()[:, None] * 1e6 ** (-2 * i / d)
        st["rope"] = torch.stack([a.cos(), a.sin()], -1).float()
        return st
    lens = _lens(c)
    st["kv_len"] = _int32(lens)
    G = math.gcd(k_h, v_h)
    if c["kind"].endswith("8"):
        st["cache"] = _cache8(g, c, lens)
    else:
        st["k"], st["v"] = (_randn(g, b, h, L, d).to(dt) for h in (k_h, v_h))
    if c["kind"].startswith("evict"):
        # what positions gather: most of them little, some much, and a part nothing at all
        w = torch.exp(3 * _randn(g, b, G, L)) * (torch.rand(b, G, L, generator=g, device=DEV) < 0.6)
        st["weights"] = w.masked_fill(torch.arange(L, device=DEV) >= st["kv_len"][:, None, None], 0.0)
        keep = c["keep"]
        st["w_out"] = torch.zeros(b, G, keep, device=DEV)
        if c["kind"] == "evict8":
            st["out"] = _empty8(c, keep)
            st["pos"] = torch.arange(keep, dtype=torch.int32, device=DEV).repeat(b)
            st["batch"] = torch.arange(b, dtype=torch.int32, device=DEV).repeat_interleave(keep)
        else:
            st["k_out"], st["v_out"] = (torch.zeros(b, h, keep, d, dtype=dt, device=DEV) for h in (k_h, v_h))
        return st
    st["q"] = _randn(g, b, q_h, 1, d).to(dt)
    st["weights"] = torch.zeros(b, G, L, device=DEV)
    st["mask"] = None
    if c["mask"]:    # left padding: row i hides its first i / 16 positions
        st["mask"] = torch.zeros(b, 1, 1, L, dtype=dt, device=DEV)
        for i in range(b):
            st["mask"][i, ..., : lens[i] * i // (16 * b)] = torch.finfo(dt).min
    return st


# ------------------------------------------------------------------- one pass

def _run_own(st):
    from saga_amd import ops
    c = st["case"]
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    norms = {name: st.get(name) for name in ("q_norm", "k_norm")}
    if c["kind"] == "norm":
        q = ops.norm_rope_kv_append(st["qkv"], q_h, st["rope"], st["pos"], st["k"], st["v"], eps=EPS, batch=st["batch"], **norms)
        return {"q": q, "k": st["k"], "v": st["v"]}
    if c["kind"] == "trace":
        return ops.attention_weights(st["q"], st["k"], st["weights"], attention_mask=st["mask"], kv_len=st["kv_len"], add=False)
    if c["kind"] == "evict":
        kept = ops.evict_kv(st["k"], st["v"], st["weights"], st["kv_len"], c["keep"], c["recent"],
                            out=(st["k_out"], st["v_out"], st["w_out"]))
        return {"kept": kept, "k": st["k_out"], "v": st["v_out"], "weights": st["w_out"]}
    cache = ops.KVFP8(**st["cache"], block=c["block"])
    if c["kind"] == "norm8":
        q = ops.norm_rope_kv_append_fp8(st["qkv"], q_h, st["rope"], st["start"], cache, eps=EPS, offsets=st["offsets"], **norms)
        k, v = ops.read_kv_fp8(cache, st["pos"], batch=st["batch"], dtype=st["qkv"].dtype)
        return {"q": q, "k": k, "v": v}
    if c["kind"] == "evict8":
        out = ops.KVFP8(**st["out"], block=c["block"])
        kept = ops.evict_kv_fp8(cache, st["weights"], st["kv_len"], c["keep"], c["recent"], out=(out, st["w_out"]))
        k, v = ops.read_kv_fp8(out, st["pos"], batch=st["batch"], dtype=DTYPES[c["dtype"]])
        return {"kept": kept, "k": k, "v": v, "weights": st["w_out"]}
    if not c["trace"]:
        return ops.dense_decode_fp8(st["q"], cache, attention_mask=st["mask"], kv_len=st["kv_len"])
    out = ops.dense_decode_fp8(st["q"], cache, attention_mask=st["mask"], kv_len=st["kv_len"], weights=st["weights"],
                               weights_add=False)
    return {"out": out, "weights": st["weights"]}


def _norm_rope(st, dtype):
    """Queries and keys normed and turned, and values, [n, heads, d] in `dtype`."""
    q_h, k_h, v_h, d = HEADS[st["case"]["heads"]]
    x = st["qkv"].to(dtype).unflatten(-1, (-1, d))
    q, k, v = x.split([q_h, k_h, v_h], 1)
    cs, sn = (st["rope"][:, None, :, i].to(dtype) for i in (0, 1))

    def turned(t, w):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w.to(dtype)
        a, b = t[..., : d // 2], t[..., d // 2:]
        return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)

    return turned(q, st["q_norm"]), turned(k, st["k_norm"]), v


def _append8(st, name, new):
    """The rows new [n, heads, d] into the 8-bit cache; what is held of them."""
    cache, block = st["cache"], st["case"]["block"]
    codes, scales = cache[name + "_codes"], cache[name + "_scales"]
    b, h, L, d = codes.shape
    nb = scales.shape[-1]
    rows, slots, start = st["batch"].long(), st["pos"].long(), st["start"].long()
    at = rows * nb + slots // block
    top = torch.zeros(b * nb, h, dtype=new.dtype, device=DEV)
    top = top.scatter_reduce(0, at[:, None].expand(-1, h), new.abs().amax(-1), "amax")
    every = torch.arange(b, device=DEV)
    touched, open_ = (torch.zeros(b * nb, 1, dtype=torch.bool, device=DEV) for _ in range(2))
    touched[at] = True
    open_[every * nb + start.clamp(max=L - 1) // block, 0] = start % block != 0
    old = scales.transpose(1, 2).reshape(b * nb, h).to(new.dtype)
    s = torch.where(touched & ~(open_ & (top <= 448 * old)), _scale(top), old)
    # what the rows' first blocks hold, at the new scales
    blk = start.clamp(max=L - 1) // block
    idx = blk[:, None] * block + torch.arange(block, device=DEV)
    live = (idx < start[:, None])[:, None, :, None]
    idx = idx.clamp(max=L - 1)
    held = codes[every[:, None, None], torch.arange(h, device=DEV)[:, None], idx[:, None]]
    s0, s1 = (t[every * nb + blk][:, :, None, None] for t in (old, s))
    again = _codes(_e4m3(_over(_open(held, new.dtype) * s0, s1)))
    codes[every[:, None, None], torch.arange(h, device=DEV)[:, None], idx[:, None]] = torch.where(live, again, held)
    scales.copy_(s.reshape(b, nb, h).transpose(1, 2))
    mine = s[at][..., None]
    c = _codes(_e4m3(_over(new, mine)))
    codes[rows, :, slots] = c
    return (_open(c) * mine.float()).to(st["qkv"].dtype)


def _kept(weights, n, keep, recent):
    """Old slots of the kept positions [b, G, keep]: heavy ones that lie below keep - recent stay, the others fill the
    gaps in order, the last `recent` positions follow; -1 behind a row's end."""
    b, G, L = weights.shape
    H = keep - recent
    p = torch.arange(max(L, keep), device=DEV)
    n = n.long()[:, None, None]
    w = torch.nn.functional.pad(weights, (0, max(L, keep) - L))
    w = w.masked_fill(p >= n - recent, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    heavy = torch.zeros_like(w, dtype=torch.bool).scatter(-1, order[..., :H], True)
    moves = heavy & (p >= H)
    gap = ~heavy & (p < H)
    at = torch.where(moves, moves.cumsum(-1) - 1, w.shape[-1])   # the i-th of those that move
    movers = torch.zeros(b, G, w.shape[-1] + 1, dtype=torch.long, device=DEV).scatter(-1, at, p.expand(b, G, -1))
    filled = movers.gather(-1, (gap.cumsum(-1) - 1).clamp(min=0))
    kept = torch.where(p >= H, n - keep + p, torch.where(gap, filled, p))[..., :keep]
    whole = torch.where(p < n, p, -1)[..., :keep]
    return torch.where(n > keep, kept, whole.expand(b, G, -1))


def _rows(t, kept, h):
    """Rows [b, heads, keep, d] of t [b, heads, L, d] at the kept slots of each head's group (slot 0 where there is none)."""
    at = kept.clamp(min=0).repeat_interleave(h // kept.shape[1], 1)
    return t.gather(2, at[..., None].expand(-1, -1, -1, t.shape[-1]))


def run(state):
    if own:
        return _run_own(state)
    st, c = state, state["case"]
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    b, L, dt = c["b"], c["L"], DTYPES[c["dtype"]]
    if c["kind"] == "norm":
        q, k, v = _norm_rope(st, torch.float32)
        rows = st["batch"].long() if st["batch"] is not None else torch.arange(b, device=DEV)
        st["k"][rows, :, st["pos"].long()] = k.to(dt)
        st["v"][rows, :, st["pos"].long()] = v.to(dt)
        return {"q": q.to(dt), "k": st["k"], "v": st["v"]}
    if c["kind"] == "norm8":   # keys in 64 bits: a rounding to 4 bits of mantissa has borders that 32 bits move across
        q, k, v = _norm_rope(st, torch.float64)
        return {"q": q.to(dt), "k": _append8(st, "k", k), "v": _append8(st, "v", v)}
    if c["kind"].startswith("evict"):
        kept = _kept(st["weights"], st["kv_len"], c["keep"], c["recent"])
        there = kept >= 0
        st["w_out"].copy_(st["weights"].gather(-1, kept.clamp(min=0)) * there)
        if c["kind"] == "evict":
            for name, h in (("k", k_h), ("v", v_h)):
                live = there.repeat_interleave(h // there.shape[1], 1)[..., None]
                st[name + "_out"].copy_(torch.where(live, _rows(st[name], kept, h), st[name + "_out"]))
            return {"kept": kept.int(), "k": st["k_out"], "v": st["v_out"], "weights": st["w_out"]}
        out = {"kept": kept.int(), "weights": st["w_out"]}
        for name, h in (("k", k_h), ("v", v_h)):
            at = kept.clamp(min=0).repeat_interleave(h // kept.shape[1], 1)
            live = there.repeat_interleave(h // there.shape[1], 1)
            s = st["cache"][name + "_scales"].gather(-1, at // c["block"]) * live
            nb = -(-c["keep"] // c["block"])
            top = torch.nn.functional.pad(s, (0, nb * c["block"] - c["keep"])).unflatten(-1, (nb, -1)).amax(-1)
            mine = top.repeat_interleave(c["block"], -1)[..., : c["keep"]]
            x = _open(_rows(st["cache"][name + "_codes"], kept, h)) * (s / torch.where(mine > 0, mine, torch.ones_like(mine)))[..., None]
            codes = torch.where(live[..., None], _codes(_e4m3(x)), st["out"][name + "_codes"])
            st["out"][name + "_codes"].copy_(codes)
            st["out"][name + "_scales"].copy_(top)
            out[name] = (_open(codes) * mine[..., None]).to(dt).transpose(1, 2).flatten(0, 1)
        return out
    if c["kind"] == "dense8":
        k = _values(st["cache"]["k_codes"], st["cache"]["k_scales"], c["block"])
    else:
        k = st["k"].float()
    x = (st["q"].float().reshape(b, k_h, q_h // k_h, d) @ k.transpose(-1, -2)).reshape(b, q_h, 1, L) / math.sqrt(d)
    if st["mask"] is not None:
        x = x + st["mask"].float()
    x = x.masked_fill(torch.arange(L, device=DEV) >= st["kv_len"][:, None, None, None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    w = p.reshape(b, math.gcd(k_h, v_h), -1, L).sum(2)
    if c["kind"] == "trace":
        return w
    v = _values(st["cache"]["v_codes"], st["cache"]["v_scales"], c["block"])
    o = (p.reshape(b, v_h, q_h // v_h, L) @ v).reshape(b, q_h, 1, d).to(dt)
    return {"out": o, "weights": w} if c["trace"] else o


# ------------------------------------------------------------------- the definition in 64 bits

def _exact_scale(top):
    """2^(floor(log2(top)) - 5) by the exponent bits of a 64-bit number."""
    e = (top.double().view(torch.int64) >> 52) - 1023
    s = (((e - 5).clamp(min=-100) + 1023) << 52).view(torch.float64)
    return torch.where(top > 0, s, torch.zeros_like(s))


def _exact_e4m3(x):
    """The nearest e4m3 number by search among all of them, ties to the even code."""
    grid = torch.arange(127, dtype=torch.uint8, device=DEV).view(F8).double()   # 0 .. 448 by code
    a = x.abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp(1, 126)
    lo = hi - 1
    under, over = a - grid[lo], grid[hi] - a
    up = (over < under) | ((over == under) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[lo]) * torch.sign(x)


def _exact_append(c, st, name, new):
    """What an append of new [n, heads, d] (float64) leaves in its own slots, a batch row and a block at a time."""
    block, got = c["block"], torch.zeros_like(new)
    start, rows = st["start"].tolist(), st["batch"].tolist()
    first = 0
    for i in range(c["b"]):
        n = rows.count(i)
        at = 0
        while at < n:
            slot = start[i] + at
            m = min(block - slot % block, n - at)
            x = new[first + at: first + at + m]
            top = x.abs().amax((0, 2))
            s = _exact_scale(top)
            if slot % block:
                old = st["cache"][name + "_scales"][i, :, slot // block].double()
                s = torch.where(top <= 448 * old, old, s)
            by = torch.where(s > 0, s, torch.ones_like(s))[None, :, None]
            got[first + at: first + at + m] = _exact_e4m3(x / by) * s[None, :, None]
            at += m
        first += n
    return got


def _exact_kept(w, n, keep, recent):
    """Kept slots of one row of weights, position by position on the host."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    H = keep - recent
    heavy = sorted(range(n - recent), key=lambda p: (-w[p], p))[:H]
    movers = iter(sorted(p for p in heavy if p >= H))
    stay = {p for p in heavy if p < H}
    return [p if p in stay else next(movers) for p in range(H)] + list(range(n - recent, n))


def exact(case, seed):
    c, st = case, prepare(case, seed)
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    b, L = c["b"], c["L"]
    if c["kind"] in ("norm", "norm8"):
        x = st["qkv"].double().unflatten(-1, (-1, d))
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        w = torch.cat([st["q_norm"].double().expand(q_h, d), st["k_norm"].double().expand(k_h, d)])
        t = (x * r)[:, : q_h + k_h] * w
        z = torch.complex(t[..., : d // 2], t[..., d // 2:]) * torch.view_as_complex(st["rope"].double())[:, None]
        y = torch.cat([z.real, z.imag], -1)
        q, k, v = y[:, :q_h], y[:, q_h:], x[:, q_h + k_h:]
        if c["kind"] == "norm8":
            return {"q": q, "k": _exact_append(c, st, "k", k), "v": _exact_append(c, st, "v", v)}
        out, pos = {"q": q}, st["pos"].tolist()
        rows = range(b) if st["batch"] is None else st["batch"].tolist()
        for name, new in (("k", k), ("v", v)):
            out[name] = st[name].double()
            for i, row in enumerate(rows):
                out[name][row, :, pos[i]] = new[i]
        return out
    if c["kind"].startswith("evict"):
        lens, w = st["kv_len"].tolist(), st["weights"].cpu().tolist()
        kept = torch.tensor([[_exact_kept(row, lens[i], c["keep"], c["recent"]) for row in w[i]] for i in range(b)], device=DEV)
        G, keep = kept.shape[1], c["keep"]
        out = {"kept": kept.int(), "weights": torch.zeros(b, G, keep, dtype=torch.float64, device=DEV)}
        for name, h in (("k", k_h), ("v", v_h)):
            got = torch.zeros(b, h, keep, d, dtype=torch.float64, device=DEV)
            for i in range(b):
                m = min(lens[i], keep)
                for j in range(h):
                    at = kept[i, j * G // h, :m]
                    out["weights"][i, j * G // h, :m] = st["weights"][i, j * G // h, at].double()
                    if c["kind"] == "evict":
                        got[i, j, :m] = st[name][i, j, at].double()
                        continue
                    codes = _open(st["cache"][name + "_codes"][i, j, at], torch.float64)
                    s = st["cache"][name + "_scales"][i, j, at // c["block"]].double()
                    for p in range(0, m, c["block"]):
                        x, t = codes[p: p + c["block"]] * s[p: p + c["block"], None], s[p: p + c["block"]].amax()
                        got[i, j, p: p + c["block"]][: x.shape[0]] = _exact_e4m3(x / t) * t if t > 0 else 0.0
            out[name] = got if c["kind"] == "evict" else got.transpose(1, 2).flatten(0, 1)
        return out
    G = math.gcd(k_h, v_h)
    w = torch.zeros(b, G, L, dtype=torch.float64, device=DEV)
    out = torch.empty(b, q_h, 1, d, dtype=torch.float64, device=DEV)
    for i in range(b):
        n = int(st["kv_len"][i])
        if c["kind"] == "dense8":
            k, v = (_values(st["cache"][s + "_codes"][i, :, :n], st["cache"][s + "_scales"][i], c["block"], torch.float64)
                    for s in "kv")
        else:
            k, v = st["k"][i, :, :n].double(), None
        for h in range(q_h):
            x = torch.mv(k[h * k_h // q_h], st["q"][i, h, 0].double()) / math.sqrt(d)
            if st["mask"] is not None:
                x = x + st["mask"][i, 0, 0, :n].double()
            p = torch.softmax(x, 0)
            w[i, h * G // q_h, :n] += p
            if v is not None:
                out[i, h, 0] = p @ v[h * v_h // q_h]
    if c["kind"] == "trace":
        return w
    return {"out": out, "weights": w} if c["trace"] else out


# ------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    b = c["b"]
    if c["kind"] in ("norm", "norm8"):   # the projection and the rotations read, queries and cache rows written
        n = (c["n"] or b) if c["kind"] == "norm" else sum(_prompt_lens(c)) if c["n"] else b
        rows = 2 if c["kind"] == "norm" else 1 + 1 + 2   # 8 bits: written, read back, and written out
        return {"bytes": n * (2 * (q_h + k_h + v_h) * d + 2 * q_h * d + 4 * d + 4 + rows * (k_h + v_h) * d),
                "flops": n * (10 * (q_h + k_h) + 4 * (k_h + v_h)) * d}
    total = sum(_lens(c))
    G = math.gcd(k_h, v_h)
    if c["kind"].startswith("evict"):
        rows = sum(min(n, c["keep"]) for n in _lens(c))
        size = 2 + 2 if c["kind"] == "evict" else 1 + 1 + 1 + 2   # read and written; 8 bits: read back and written out
        return {"bytes": 4 * G * (total + b * c["keep"] + rows) + size * rows * (k_h + v_h) * d, "flops": G * total}
    if c["kind"] == "trace":
        return {"bytes": 2 * total * k_h * d + 2 * b * q_h * d + 4 * b * G * c["L"], "flops": 2 * total * q_h * d}
    return {"bytes": total * (k_h + v_h) * d + 4 * (total // c["block"]) * (k_h + v_h) + 4 * b * q_h * d
            + (2 * total if c["mask"] else 0) + (4 * b * G * c["L"] if c["trace"] else 0),
            "flops": 4 * total * q_h * d}
