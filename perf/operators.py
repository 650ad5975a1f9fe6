"""Operators on data held in 4 bits, on one MI355X: decode projections with 4-bit weights, such weights opened for a
prompt's products, rotary embedding with the append to a 4-bit key / value cache, rows read back from it, and decode
attention over it.

Values are s * c + z: codes c of 4 bits, and per group of consecutive values one scale s and one offset z in f16.
`own` False computes the plain form in elementary torch operations from the same packed buffers; True calls saga_amd.

Head layouts and widths are those of the decoder shapes in saga_amd/decoder.py (12 query / 1 key / 2 value heads of
128, and 15 / 1 / 5 of 64, each also with as many key heads as value heads); lengths, batches and positions are those
of bench.py and of the latency grid of saga_amd/speedup.py (batch 1-32, 4k-64k positions).
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
# query, key and value heads, head dim
HEADS = {"12/1/2x128": (12, 1, 2, 128), "12/2/2x128": (12, 2, 2, 128), "15/1/5x64": (15, 1, 5, 64),
         "15/5/5x64": (15, 5, 5, 64)}
# rows and columns of the decode projections, their epilogues, whether the input's RMSNorm is fused
PROJ = {"qkv": (1920, 1536, "bias", True), "o": (1536, 1536, "store", False),
        "gate_up": (17920, 1536, "silu_pairs", True), "down": (1536, 8960, "store", False),
        "head": (151936, 1536, "store", True), "small_o": (960, 960, "store", False),
        "small_gate_up": (5120, 960, "silu_pairs", True), "small_down": (960, 2560, "store", False)}


def listed():
    return [
        # One token of the smallest model, output projection: the least work of a decode step, a launch's latency.
        {"name": "gemv_b1_small_o", "kind": "gemv", "proj": "small_o", "m": 1, "group": 32},
        # Gate / up projection with RMSNorm and SiLU at the headline batch: most of a decode step's weight bytes.
        {"name": "gemv_b8_gate_up", "kind": "gemv", "proj": "gate_up", "m": 8, "group": 64},
        # Down projection, long rows and few of them, an odd batch, the usual group of 4-bit checkpoints.
        {"name": "gemv_b5_down", "kind": "gemv", "proj": "down", "m": 5, "group": 128},
        # The LM head at the largest batch that the skinny product takes.
        {"name": "gemv_b32_head", "kind": "gemv", "proj": "head", "m": 32, "group": 64},
        # Weights opened for a prompt's matrix products: a small layer's, and the widest of the headline model.
        {"name": "unpack_small_down", "kind": "unpack", "proj": "small_down", "group": 32},
        {"name": "unpack_gate_up", "kind": "unpack", "proj": "gate_up", "group": 64},
        # A decode step's new tokens into the cache, each at its own position, and their rows read back.
        {"name": "append_b8", "kind": "append", "heads": "12/1/2x128", "b": 8, "n": 0, "L": 33024, "group": 64,
         "dtype": "bf16"},
        # A prompt's tokens into one batch row, and all of them read back for its attention.
        {"name": "append_prompt_4001", "kind": "append", "heads": "12/1/2x128", "b": 8, "n": 4001, "L": 4352,
         "group": 32, "dtype": "bf16"},
        # One sequence of the small model over a short cache: latency.
        {"name": "dense_b1_4k", "kind": "dense", "heads": "15/1/5x64", "b": 1, "L": 4096, "fill": 4096, "group": 32,
         "dtype": "bf16", "mask": False},
        # The headline decode's attention: static cache, 32769 filled positions.
        {"name": "dense_b8_32k", "kind": "dense", "heads": "12/1/2x128", "b": 8, "L": 33024, "fill": 32769, "group": 64,
         "dtype": "bf16", "mask": False},
        # A served batch of different lengths with left padding masked off, plain GQA, f16.
        {"name": "dense_b4_8k_ragged", "kind": "dense", "heads": "15/5/5x64", "b": 4, "L": 8195, "fill": 0, "group": 64,
         "dtype": "f16", "mask": True},
        # The largest cell of the latency grid: batch 32 at 64k positions.
        {"name": "dense_b32_64k", "kind": "dense", "heads": "12/1/2x128", "b": 32, "L": 65544, "fill": 65541,
         "group": 32, "dtype": "bf16", "mask": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gemv", "gemv", "gemv", "unpack", "append", "append", "dense", "dense", "dense"])
    if kind in ("gemv", "unpack"):
        name = rng.choice([p for p in PROJ if kind == "gemv" or p != "head"])
        c = {"kind": kind, "proj": name, "group": rng.choice([g for g in (32, 64, 128) if PROJ[name][1] % g == 0])}
        if kind == "gemv":
            c["m"] = _log(rng, 1, 32)
        return c
    c = {"kind": kind, "heads": rng.choice(list(HEADS)), "group": rng.choice([32, 64]),
         "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "append":
        c["b"] = _log(rng, 1, 32)
        c["n"] = rng.choice([0, _log(rng, 2, 4000)])
        c["L"] = max(c["n"], 1) + _log(rng, 100, 4000)
    else:
        c["b"] = _log(rng, 1, 32)
        c["L"] = _log(rng, 100, min(65000, 1000000 // c["b"]))
        c["fill"] = rng.choice([0, c["L"], max(1, c["L"] - c["L"] // 50)])
        c["mask"] = rng.random() < 0.25
    return c


# ------------------------------------------------------------------- the 4-bit form
# Codes' places. Keys: word s * (d / 32) + j of a row holds dims 32 j + 8 s + e, e-th nibble. Values: nibble e of the
# c-th of 16 units of d / 16 nibbles is dim 16 e + c. Weights: unit [16 rows][128 columns] of 64 lanes of 4 words, word j
# of lane 16 s + c is row c at columns 32 j + 8 s + (0, 2, 4, 6, 1, 3, 5, 7), nibble by nibble.

def _f16_down(x):
    """The largest f16 that is at most x (x at most 65504 in magnitude)."""
    h = x.to(torch.float16)
    bits = h.view(torch.int16)
    under = torch.where(bits > 0, bits - 1, torch.where(bits == 0, torch.full_like(bits, -32767), bits + 1))
    return torch.where(h.to(x.dtype) > x, under, bits).view(torch.float16)


def _f16_up(x):
    return -_f16_down(-x)


def _quantise(x, group):
    """Codes (uint8, x's shape) and [..., n / group, 2] f16 scales and offsets of x [..., n] in its own precision."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    z = _f16_down(lo)
    s = _f16_up((hi - z.to(x.dtype)) / torch.full_like(hi, 15.0))
    c = torch.round((g - z.to(x.dtype)) / torch.where(s == 0, torch.ones_like(s), s).to(x.dtype)).clamp(0, 15)
    return c.to(torch.uint8).reshape(x.shape), torch.cat([s, z], -1)


def _dequantise(c, sz, dtype):
    g = c.reshape(*c.shape[:-1], sz.shape[-2], -1).to(dtype)
    return (g * sz[..., :1].to(dtype) + sz[..., 1:].to(dtype)).reshape(c.shape)


def _nibbles(c):
    """Nibbles [..., 2 n] (the first in the low half of a byte) to bytes [..., n]."""
    p = c.reshape(*c.shape[:-1], -1, 2)
    return p[..., 0] | (p[..., 1] << 4)


def _open(b):
    return torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def _pack_k(c):
    d = c.shape[-1]
    return _nibbles(c.reshape(*c.shape[:-1], d // 32, 4, 8).transpose(-2, -3).reshape(c.shape))


def _open_k(b):
    c = _open(b)
    return c.reshape(*c.shape[:-1], 4, c.shape[-1] // 32, 8).transpose(-2, -3).reshape(c.shape)


def _pack_v(c):
    return _nibbles(c.reshape(*c.shape[:-1], -1, 16).transpose(-1, -2).reshape(c.shape))


def _open_v(b):
    c = _open(b)
    return c.reshape(*c.shape[:-1], 16, -1).transpose(-1, -2).reshape(c.shape)


def _pack_w(c):
    n, k = c.shape
    c = torch.nn.functional.pad(c, (0, -k % 128))
    c = c.reshape(n // 16, 16, -1, 4, 4, 4, 2)              # tile, row, unit, word, lane group, pair, half
    return _nibbles(c.permute(0, 2, 4, 1, 3, 6, 5).reshape(n // 16, -1, 2048))


def _open_w(b, k):
    c = _open(b).reshape(b.shape[0], b.shape[1], 4, 16, 4, 2, 4)
    return c.permute(0, 3, 1, 4, 2, 6, 5).reshape(16 * b.shape[0], -1)[:, :k]


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device=DEV, dtype=dtype)


def _layout(c):
    q_h, k_h, v_h, d = HEADS[c["heads"]]
    return q_h, k_h, v_h, d, d // c["group"]


def _cache(b, k_h, v_h, L, d, ng):
    return {"k_codes": torch.zeros(b, k_h, L, d // 2, dtype=torch.uint8, device=DEV),
            "k_scales": torch.zeros(b, k_h, L, 2 * ng, dtype=torch.float16, device=DEV),
            "v_codes": torch.zeros(b, v_h, L, d // 2, dtype=torch.uint8, device=DEV),
            "v_scales": torch.zeros(b, v_h, L, 2 * ng, dtype=torch.float16, device=DEV)}


def prepare(case, seed):
    c, g = case, _gen(seed)
    st = {"case": c}
    if c["kind"] in ("gemv", "unpack"):
        n, k, epilogue, rms = PROJ[c["proj"]]
        codes, scales = [], []
        for r0 in range(0, n, 16384):
            cc, sz = _quantise(0.03 * _randn(g, min(16384, n - r0), k), c["group"])
            codes.append(_pack_w(cc))
            scales.append(sz.reshape(-1, 16, k // c["group"], 2).transpose(1, 2).contiguous())
        st["codes"], st["scales"] = torch.cat(codes), torch.cat(scales)
        if c["kind"] == "gemv":
            st["x"] = _randn(g, c["m"], k).to(torch.bfloat16)
            st["bias"] = _randn(g, n).to(torch.bfloat16) if epilogue == "bias" else None
        return st
    q_h, k_h, v_h, d, ng = _layout(c)
    b, L, dt = c["b"], c["L"], DTYPES[c["dtype"]]
    st["cache"] = _cache(b, k_h, v_h, L, d, ng)
    if c["kind"] == "append":
        n = c["n"] or b
        st["qkv"] = _randn(g, n, (q_h + k_h + v_h) * d).to(dt)
        if c["n"]:   # a prompt into batch row b - 1, behind whatever of it is there
            st["pos"] = torch.arange(n, dtype=torch.int32, device=DEV) + (L - n) // 2
            st["batch"] = torch.full((n,), b - 1, dtype=torch.int32, device=DEV)
        else:        # one token of every batch row
            st["pos"] = torch.randint(L // 2, L, (n,), generator=g, device=DEV, dtype=torch.int32)
            st["batch"] = None
        i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
        a = st["pos"].double()[:, None] * 1e6 ** (-2 * i / d)
        st["rope"] = torch.stack([a.cos(), a.sin()], -1).float()
        return st
    lens = [c["fill"]] * b if c["fill"] else [L - (3 * L // 4) * i // b for i in range(b)]
    st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["q"] = _randn(g, b, q_h, 1, d).to(dt)
    outlier = 1 + 3 * (torch.rand(d, generator=g, device=DEV) < 0.05)   # keys have a few long dims
    for i in range(b):
        for h, pack, name, by in ((k_h, _pack_k, "k", outlier), (v_h, _pack_v, "v", 1)):
            x = _randn(g, h, lens[i], d) * by
            cc, sz = _quantise(x, c["group"])
            st["cache"][name + "_codes"][i, :, :lens[i]] = pack(cc)
            st["cache"][name + "_scales"][i, :, :lens[i]] = sz.flatten(-2)
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
    if c["kind"] in ("gemv", "unpack"):
        w = ops.Q4Weight(st["codes"], st["scales"], c["group"])
        if c["kind"] == "unpack":
            return ops.unpack_gemv_q4([w])[0]
        _, _, epilogue, rms = PROJ[c["proj"]]
        return ops.gemv_q4(st["x"], w, bias=st["bias"], rms_eps=EPS if rms else None,
                           epilogue="silu_pairs" if epilogue == "silu_pairs" else "store")
    cache = ops.KVQ4(**st["cache"])
    if c["kind"] == "append":
        q = ops.rope_kv_append_q4(st["qkv"], HEADS[c["heads"]][0], st["rope"], st["pos"], cache, batch=st["batch"])
        k, v = ops.read_kv_q4(cache, st["pos"], batch=st["batch"], dtype=st["qkv"].dtype)
        return {"q": q, "k": k, "v": v}
    return ops.dense_decode_q4(st["q"], cache, attention_mask=st["mask"], kv_len=st["kv_len"])


def _weight(st, dtype):
    sz = st["scales"].transpose(1, 2).flatten(0, 1)
    return _dequantise(_open_w(st["codes"], sz.shape[1] * st["case"]["group"]), sz, dtype)


def _rows(t, name, ng, dtype, opened):
    sz = t[name + "_scales"].unflatten(-1, (ng, 2))
    return _dequantise(opened(t[name + "_codes"]), sz, dtype)


def run(state):
    if own:
        return _run_own(state)
    st, c = state, state["case"]
    if c["kind"] == "unpack":
        return _weight(st, torch.float32).to(torch.bfloat16)
    if c["kind"] == "gemv":
        _, _, epilogue, rms = PROJ[c["proj"]]
        x = st["x"].float()
        if rms:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        y = x @ _weight(st, torch.float32).t()
        if epilogue == "bias":
            y = y + st["bias"].float()
        if epilogue == "silu_pairs":
            y = y[:, 0::2] / (1 + torch.exp(-y[:, 0::2])) * y[:, 1::2]
        return y.to(torch.bfloat16)
    q_h, k_h, v_h, d, ng = _layout(c)
    if c["kind"] == "append":
        n, dt = st["qkv"].shape[0], st["qkv"].dtype
        x = st["qkv"].reshape(n, q_h + k_h + v_h, d).float()
        cs, sn = st["rope"][:, None, :, 0], st["rope"][:, None, :, 1]
        x1, x2 = x[:, : q_h + k_h, : d // 2], x[:, : q_h + k_h, d // 2:]
        y = torch.cat([x1 * cs - x2 * sn, x2 * cs + x1 * sn], -1)
        rows = st["batch"].long() if st["batch"] is not None else torch.arange(n, device=DEV)
        pos = st["pos"].long()
        out = {"q": y[:, :q_h].to(dt)}
        for name, new, pack, opened in (("k", y[:, q_h:], _pack_k, _open_k), ("v", x[:, q_h + k_h:], _pack_v, _open_v)):
            codes, sz = _quantise(new, c["group"])
            st["cache"][name + "_codes"][rows, :, pos] = pack(codes)
            st["cache"][name + "_scales"][rows, :, pos] = sz.flatten(-2)
            held = {f"{name}_{p}": st["cache"][f"{name}_{p}"][rows, :, pos] for p in ("codes", "scales")}
            out[name] = _rows(held, name, ng, torch.float32, opened).to(dt)
        return out
    b, L = c["b"], c["L"]
    k = _rows(st["cache"], "k", ng, torch.float32, _open_k)
    v = _rows(st["cache"], "v", ng, torch.float32, _open_v)
    x = (st["q"].float().reshape(b, k_h, q_h // k_h, d) @ k.transpose(-1, -2)).reshape(b, q_h, 1, L) / math.sqrt(d)
    if st["mask"] is not None:
        x = x + st["mask"].float()
    x = x.masked_fill(torch.arange(L, device=DEV) >= st["kv_len"][:, None, None, None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).reshape(b, v_h, q_h // v_h, L)
    return (p @ v).reshape(b, q_h, 1, d).to(st["q"].dtype)


# ------------------------------------------------------------------- the definition in 64 bits

def _exact_values(x, group):
    """What x (float64) is held as: per group z the largest f16 <= min, s the smallest f16 >= (max - z) / 15."""
    g = x.reshape(*x.shape[:-1], -1, group)
    z = _f16_down(g.amin(-1, keepdim=True)).double()
    s = _f16_up((g.amax(-1, keepdim=True) - z) / 15.0).double()
    steps = torch.where(s > 0, (g - z) / s, torch.zeros_like(g))
    return (z + s * torch.round(steps).clamp(0, 15)).reshape(x.shape)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] in ("gemv", "unpack"):
        group = c["group"]
        codes, sz = _open_w(st["codes"], st["scales"].shape[1] * group), st["scales"].double()
        n, k = codes.shape
        s = sz[..., 0].permute(0, 2, 1).reshape(n, -1).repeat_interleave(group, 1)
        z = sz[..., 1].permute(0, 2, 1).reshape(n, -1).repeat_interleave(group, 1)
        w = s.mul_(codes).add_(z)
        if c["kind"] == "unpack":
            return w
        _, _, epilogue, rms = PROJ[c["proj"]]
        x = st["x"].double()
        if rms:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        y = torch.mm(x, w.t())
        if epilogue == "bias":
            y = y + st["bias"].double()
        if epilogue == "silu_pairs":
            gate, up = y[:, 0::2], y[:, 1::2]
            y = gate * torch.sigmoid(gate) * up
        return y
    q_h, k_h, v_h, d, ng = _layout(c)
    if c["kind"] == "append":
        x = st["qkv"].double().unflatten(-1, (-1, d))
        rot = torch.view_as_complex(st["rope"].double())[:, None]
        z = torch.complex(x[..., : d // 2], x[..., d // 2:])[:, : q_h + k_h] * rot
        y = torch.cat([z.real, z.imag], -1)
        return {"q": y[:, :q_h], "k": _exact_values(y[:, q_h:], c["group"]),
                "v": _exact_values(x[:, q_h + k_h:], c["group"])}
    out = torch.empty(c["b"], q_h, 1, d, dtype=torch.float64, device=DEV)
    for i in range(c["b"]):
        n = int(st["kv_len"][i])
        held = {name: t[i, :, :n] for name, t in st["cache"].items()}
        k, v = _rows(held, "k", ng, torch.float64, _open_k), _rows(held, "v", ng, torch.float64, _open_v)
        for h in range(q_h):
            x = torch.mv(k[h * k_h // q_h], st["q"][i, h, 0].double()) / math.sqrt(d)
            if st["mask"] is not None:
                x = x + st["mask"][i, 0, 0, :n].double()
            out[i, h, 0] = torch.softmax(x, 0) @ v[h * v_h // q_h]
    return out


# ------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] in ("gemv", "unpack"):
        n, k, epilogue, _ = PROJ[c["proj"]]
        held = n * k // 2 + n * (k // c["group"]) * 4
        if c["kind"] == "unpack":
            return {"bytes": held + 2 * n * k, "flops": 2 * n * k}
        outs = n // 2 if epilogue == "silu_pairs" else n
        return {"bytes": held + 2 * c["m"] * (k + outs) + (2 * n if epilogue == "bias" else 0), "flops": 2 * c["m"] * n * k}
    q_h, k_h, v_h, d, ng = _layout(c)
    row = d // 2 + 4 * ng
    if c["kind"] == "append":   # the projection read, queries and cache rows written, those read back and written out
        n = c["n"] or c["b"]
        return {"bytes": n * (2 * (q_h + k_h + v_h) * d + 2 * q_h * d + 4 * d + 4 + 2 * (k_h + v_h) * row
                              + 2 * (k_h + v_h) * d), "flops": n * (6 * q_h + 16 * (k_h + v_h)) * d}
    L, b = c["L"], c["b"]
    total = c["fill"] * b if c["fill"] else sum(L - (3 * L // 4) * i // b for i in range(b))
    return {"bytes": total * (k_h + v_h) * row + 4 * b * q_h * d + (2 * total if c["mask"] else 0),
            "flops": 4 * total * q_h * d}
