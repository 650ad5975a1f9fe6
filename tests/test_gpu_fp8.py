"""The 8-bit cache on the GPU against 64-bit arithmetic: what an append holds, what is read back, attention over it, the
weights of its positions."""
import math

import pytest
import torch

import fp8_util as F
from saga_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}
# Below its smallest normal number a type's numbers are evenly spaced (f16: 2^-24 under 2^-14): half a step there.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _close(got, ref, tol):
    """Within tol; NaN (a row without keys) where the reference is and nowhere else."""
    bad = ~((got.double() - ref).abs() <= tol) & ~(got.isnan() & ref.isnan())
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(((got.double() - ref).abs() / tol).max()))


# ------------------------------------------------------------------- append and read

def _keys(qkv, table, n_q, n_k, d, norm, eps):
    """Keys [N, n_k, d] of the formula in 64 bits."""
    x = qkv.double().reshape(qkv.shape[0], -1, d)[:, n_q:n_q + n_k]
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    cs, sn = table[:, None, :, 0].double(), table[:, None, :, 1].double()
    a, b = x[..., : d // 2], x[..., d // 2:]
    return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)


def _append_reference(cache, k, v, start, lens):
    """The cache after rows of lens tokens at start, head by head on the CPU."""
    want = [t.cpu().clone() for t in cache[:4]]
    at = 0
    for i, (p, n) in enumerate(zip(start, lens)):
        if n and 0 <= p and p + n <= want[0].shape[2]:
            for x, codes, scales in ((k, want[0], want[1]), (v, want[2], want[3])):
                for h in range(codes.shape[1]):
                    F.append(codes[i, h], scales[i, h], cache.block, p, x[at:at + n, h].cpu())
        at += n
    return ops.KVFP8(*(t.cuda() for t in want), cache.block)


def _run_append(g, cache, start, lens, n_q, dtype, norm=True, offsets=True, scale=1.0):
    d, n_k, n_v, n = cache.k_codes.shape[-1], cache.k_codes.shape[1], cache.v_codes.shape[1], sum(lens)
    qkv = (_randn(g, n, (n_q + n_k + n_v) * d) * scale).to(dtype)
    pos = torch.cat([torch.arange(k) + p for p, k in zip(start, lens)]).int().cuda() if n else _int32([])
    table = ops.rope_table(pos.clamp(min=0), d, 1e4)
    qn, kn = ((1 + 0.3 * _randn(g, d)).to(dtype) for _ in range(2)) if norm else (None, None)
    k, v = _keys(qkv, table, n_q, n_k, d, kn, 1e-6), qkv.double().reshape(n, -1, d)[:, n_q + n_k:]
    want = _append_reference(cache, k, v, start, lens)
    off = _int32([sum(lens[:i]) for i in range(len(lens) + 1)]) if offsets else None
    q = ops.norm_rope_kv_append_fp8(qkv, n_q, table, _int32(start), cache, qn, kn, offsets=off)
    # queries as into a 16-bit cache
    kc, vc = (torch.zeros(1, h, n + 1, d, dtype=dtype, device="cuda") for h in (n_k, n_v))
    plain = ops.norm_rope_kv_append(qkv, n_q, table, torch.arange(n, device="cuda").int(), kc, vc, qn, kn,
                                    batch=torch.zeros(n, device="cuda").int())
    size = _query_size(qkv, n_q, d, qn)
    live = torch.cat([torch.full((m,), 0 <= p and p + m <= cache.k_codes.shape[2]) for p, m in zip(start, lens)]).cuda()
    assert q[~live].isnan().all()
    _close(q[live], plain[live].double(), (48 * U32 + 2 * HALF[dtype]) * size[live] + 2 * TINY[dtype])
    assert F.same(cache, want)
    return qkv, table


def _query_size(qkv, n_q, d, norm):
    """A bound of the queries' magnitudes: both partners of a rotation."""
    x = qkv.double().reshape(qkv.shape[0], -1, d)[:, :n_q]
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.double()
    a, b = x[..., : d // 2].abs(), x[..., d // 2:].abs()
    return torch.cat([a + b, a + b], -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_q,n_k,n_v,d", [(12, 1, 2, 128), (15, 1, 5, 64), (4, 4, 2, 64), (2, 1, 1, 128)])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_append_tokens_one_by_one(n_q, n_k, n_v, d, block, dtype):
    """A decode's appends over block borders, with tokens that outgrow their block's scale and tokens of zeros: codes
    and scales equal the rule bit for bit, nothing else is touched."""
    g = _gen(n_q * d + block)
    B, L = 3, 2 * block + 5
    cache = F.random_cache(g, B, n_k, n_v, L, d, block)
    start = [0, block - 3, 2 * block - 1]
    for i, scale in enumerate((1.0, 0.1, 40.0, 1.0, 0.0, 3000.0)):
        _run_append(g, cache, [p + i for p in start], [1] * B, n_q, dtype, norm=i % 2 == 0, offsets=i == 3, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_q,n_k,n_v,d", [(12, 1, 2, 128), (5, 5, 1, 64)])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_append_prompts(n_q, n_k, n_v, d, block, dtype):
    """Prompts of equal lengths, ragged ones with empty rows, behind what a block holds and over it, with growth."""
    g = _gen(n_q * d + block + 1)
    L = 5 * block + 17
    cache = F.random_cache(g, 4, n_k, n_v, L, d, block)
    _run_append(g, cache, [0, 3, block, block - 1], [2 * block + 1] * 4, n_q, dtype, offsets=False)
    _run_append(g, cache, [1, block, 7, 2 * block + 5], [3 * block + 4, 0, 1, 2], n_q, dtype, scale=30.0)
    _run_append(g, cache, [0, 0, 5 * block, 0], [0, 5 * block + 17, 17, 1], n_q, dtype, norm=False)
    few = cache.rows(1, 2)  # rows of a larger cache
    _run_append(g, few, [9, block + 40], [block, 2 * block], n_q, dtype, scale=900.0)


def test_append_many_rows():
    """More rows than a wave has lanes, most of them short or empty."""
    g, B, d, block = _gen(7), 150, 64, 32
    cache = F.random_cache(g, B, 1, 1, 100, d, block)
    lens = [(i * 7) % 5 if i % 3 else (40 if i % 9 == 0 else 0) for i in range(B)]
    _run_append(g, cache, [(i * 13) % 50 for i in range(B)], lens, 1, torch.bfloat16)


def test_append_out_of_range_rows():
    """A row that does not fit writes nothing and gives NaN queries, beside rows that do."""
    g, block = _gen(8), 32
    cache = F.random_cache(g, 4, 1, 2, 70, 64, block)
    _run_append(g, cache, [-1, 60, 65, 70], [1, 1, 1, 1], 2, torch.bfloat16, offsets=False)
    _run_append(g, cache, [-40, 60, 65, 2 ** 31 - 5], [50, 10, 6, 3], 2, torch.bfloat16)


def test_append_special_values():
    """NaN and infinities are held as NaN and set no scale; magnitudes to the ends of bf16's range read back within 2^-4."""
    g, d, block, n_q = _gen(9), 64, 32, 1
    cache = F.random_cache(g, 2, 1, 1, 64, d, block)
    qkv = _randn(g, 2 * 20, 3 * d)
    v = qkv.view(40, 3, d)[:, 2]
    v[0, 3], v[1, 5], v[2, 6] = float("nan"), float("inf"), float("-inf")
    v[20:] = 0.0
    v[20, :8] = torch.tensor([3.3e38, -3.3e38, 1e30, 1e-30, 0.0, -0.0, 2.0 ** 100, -1.0], device="cuda")
    qkv = qkv.to(torch.bfloat16)
    table = ops.rope_table(torch.arange(40, device="cuda").int(), d, 1e4)
    want = _append_reference(cache, _keys(qkv, table, 1, 1, d, None, 0), qkv.double().view(40, 3, d)[:, 2:], [0, 0], [20, 20])
    ops.norm_rope_kv_append_fp8(qkv, n_q, table, _int32([0, 0]), cache)
    assert F.same(cache, want)
    k, got = ops.read_kv_fp8(cache, _int32([0, 1, 2, 3]), batch=_int32([0] * 4), dtype=torch.float32)
    assert got[0, 0, 3].isnan() and got[1, 0, 5].isnan() and got[2, 0, 6].isnan() and got.isnan().sum() == 3
    k, got = ops.read_kv_fp8(cache, _int32([0, 64, -1]), batch=_int32([1, 1, 1]), dtype=torch.float32)
    assert got[1:].isnan().all() and k[1:].isnan().all()
    x = qkv.view(40, 3, d)[20, 2].double()
    assert ((got[0, 0].double() - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * cache.v_scales[1, 0, 0].double()).all()
    # a token of NaN alone leaves a block of zeros without a scale
    one = qkv[:1].clone()
    one[:, 2 * d:] = float("nan")
    row = cache.rows(0)
    ops.norm_rope_kv_append_fp8(one, 1, table[:1].contiguous(), _int32([32]), row)
    assert row.v_scales[0, 0, 1] == 0 and ops.read_kv_fp8(row, _int32([32]))[1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_read_all_codes(dtype):
    """All 256 bytes under several scales, in every position of a row."""
    d, block = 128, 32
    codes = (torch.arange(64 * d, device="cuda") * 5 % 256).to(torch.uint8).view(1, 1, 64, d)
    scales = torch.tensor([[[2.0 ** -3, 1.7]]], device="cuda")
    cache = ops.KVFP8(codes, scales, codes.flip(-1).contiguous(), scales * 2, block)
    pos = torch.arange(64, device="cuda").int()
    zero = torch.zeros(64, device="cuda").int()
    for got, c, s in zip(ops.read_kv_fp8(cache, pos, zero, dtype=dtype), (cache.k_codes, cache.v_codes), (scales, scales * 2)):
        want = F.values(c, s, block, torch.float32)[0, 0].to(dtype)
        assert torch.equal(got[:, 0].nan_to_num(-1.0), want.nan_to_num(-1.0))
    top = ops.KVFP8(torch.full_like(codes, 0x7e), torch.full_like(scales, 2.0 ** 8), codes, scales, block)
    assert (ops.read_kv_fp8(top, pos[:1], zero[:1], dtype=torch.float16)[0] == 65504).all()  # 448 * 256


def test_strided_caches():
    """Views: gaps between positions, heads and scales give what contiguous caches do."""
    g, block, d, L = _gen(10), 64, 128, 130
    plain = F.random_cache(g, 2, 1, 2, L, d, block)
    gaps = ops.KVFP8(*(torch.zeros(2, L, 3, d + 16, dtype=torch.uint8, device="cuda").transpose(1, 2)[:, :h, :, :d] if i % 2 == 0 else
                       torch.zeros(2, 3, 7, device="cuda")[:, :h, 2:5] for h in (1, 2) for i in range(2)), block)
    for a, b in zip(plain[:4], gaps[:4]):
        b.copy_(a)
    qkv = _randn(g, 2 * 9, 7 * d, dtype=torch.bfloat16)
    wide = torch.zeros(18, 7 * d + 5, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:-2] = qkv
    table, start = ops.rope_table(torch.arange(18, device="cuda").int(), d, 1e4), _int32([60, 119])
    q = ops.norm_rope_kv_append_fp8(qkv, 4, table, start, plain)
    q2 = ops.norm_rope_kv_append_fp8(wide[:, 3:-2], 4, table, start, gaps)
    assert torch.equal(q, q2) and all(torch.equal(a, b) for a, b in zip(plain[:4], gaps[:4]))
    pos, row = _int32([0, 64, 129]), _int32([1, 0, 1])
    assert all(torch.equal(a, b) for a, b in zip(ops.read_kv_fp8(plain, pos, row), ops.read_kv_fp8(gaps, pos, row)))
    query = _randn(g, 2, 4, 1, d, dtype=torch.bfloat16)
    wp, wg = torch.zeros(2, 1, L, device="cuda"), torch.zeros(2, 2, L + 9, device="cuda")[:, ::2]
    a = ops.dense_decode_fp8(query, plain, kv_len=_int32([L, 61]), weights=wp)
    b = ops.dense_decode_fp8(query, gaps, kv_len=_int32([L, 61]), weights=wg)
    assert torch.equal(a, b) and torch.equal(wp, wg[..., :L]) and not wg[..., L:].any()


# ------------------------------------------------------------------- attention

def _dense_ref(q, k, v, mask, kv_len, scale):
    """Attention in 64 bits, the weights per head, and bounds of the kernel's errors: a score's fp32 sums (at most 64
    roundings of its largest partial sum, and the mask's) move each weight by twice that relative, the exponential by
    2^-20; a weight's terms keep 16 bits (2^-16 of p v), sums over the positions at most L / 16 + 64 roundings."""
    b, q_h, _, d = q.shape
    L = k.shape[2]
    out, tol = (torch.empty(b, q_h, d, dtype=torch.float64, device="cuda") for _ in range(2))
    w, wtol = (torch.zeros(b, q_h, L, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        n = L if kv_len is None else min(max(int(kv_len[i]), 0), L)
        for h in range(q_h):
            kh, vh = h * k.shape[1] // q_h, h * v.shape[1] // q_h
            qd = q[i, h, 0].double()
            x = k[i, kh, :n] @ qd * scale
            e = k[i, kh, :n].abs() @ qd.abs() * scale * 64 * U32
            if mask is not None:
                m = mask[i % mask.shape[0], h % mask.shape[1], 0, :n].double()
                x = x + m
                e = e + torch.where(m.isfinite(), m.abs().clamp(max=1e6), torch.zeros_like(m)) * U32
            p = torch.softmax(x, 0)
            out[i, h] = p @ v[i, vh, :n]
            ew = (2 * float(e.max()) + 2.0 ** -20) if n else 0.0
            pv = p @ v[i, vh, :n].abs()
            tol[i, h] = 2 * ew * (pv + out[i, h].abs()) + (2.0 ** -16 + (n / 16 + 64) * U32) * pv
            w[i, h, :n] = p
            wtol[i, h, :n] = p * (2 * ew + (n / 16 + 64) * U32)
    return out[:, :, None], tol[:, :, None], w, wtol


def _check(q, cache, mask, kv, scale, G=None, rows=None):
    """Outputs in fp32 and in q's type, without and with the weights of G groups; the weights."""
    k, v = F.cache_values(cache)
    fm = None if mask is None else mask[..., : k.shape[2]].to(torch.float32) if mask.dtype == torch.bool else mask[..., : k.shape[2]]
    ref, tol, w, wtol = _dense_ref(q, k, v, fm, kv, scale)
    rows = list(range(q.shape[0])) if rows is None else rows
    call = dict(attention_mask=mask, kv_len=kv, scaling=scale)
    got = ops.dense_decode_fp8(q, cache, out_dtype=torch.float32, **call)
    _close(got[rows], ref[rows], tol[rows] + U32 * ref[rows].abs())
    _close(ops.dense_decode_fp8(q, cache, **call)[rows], ref[rows], tol[rows] + HALF[q.dtype] * (ref[rows].abs() + tol[rows]) + TINY[q.dtype])
    G = math.gcd(cache.k_codes.shape[1], cache.v_codes.shape[1]) if G is None else G
    wr, wt = (t.nan_to_num(0.0).unflatten(1, (G, -1)).sum(2) for t in (w, wtol))
    weights = torch.full((q.shape[0], G, k.shape[2]), float("nan"), device="cuda")
    again = ops.dense_decode_fp8(q, cache, out_dtype=torch.float32, weights=weights, weights_add=False, **call)
    assert torch.equal(got.view(torch.int32), again.view(torch.int32))
    _close(weights[rows], wr[rows], wt[rows] + (q.shape[1] // G) * U32 * wr[rows])
    return got, weights


LAYOUTS = [(12, 1, 2, 128), (12, 2, 2, 128), (15, 1, 5, 64), (15, 5, 5, 64), (12, 3, 2, 64), (12, 4, 1, 128), (32, 1, 2, 64),
           (6, 6, 6, 128), (16, 1, 1, 64), (24, 1, 8, 128), (1, 1, 1, 64), (12, 2, 3, 128), (40, 2, 1, 64), (16, 1, 4, 128),
           (20, 2, 20, 64), (80, 1, 1, 64)]


@pytest.mark.parametrize("q_h,k_h,v_h,d", LAYOUTS)
@pytest.mark.parametrize("dtype,block", [(torch.bfloat16, 64), (torch.bfloat16, 32), (torch.float16, 128)])
def test_dense_layouts(q_h, k_h, v_h, d, dtype, block):
    g = _gen(q_h * d + block)
    b, L = 3, 301
    cache = F.random_cache(g, b, k_h, v_h, L, d, block)
    q = _randn(g, b, q_h, 1, d, dtype=dtype)
    _check(q, cache, None, _int32([301, 1, 133]), 1 / math.sqrt(d))


@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 1000, 4099, 33000])
@pytest.mark.parametrize("b", [1, 9])
def test_dense_lengths(L, b):
    """Lengths around the steps, splits and blocks; what lies behind kv_len holds NaN."""
    g = _gen(L + b)
    q_h, k_h, v_h, d, block = 12, 1, 2, 128, 32
    cache = F.random_cache(g, b, k_h, v_h, L, d, block)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    lens = [max(1, L - (3 * L // 4) * i // b) for i in range(b)]
    kv = _int32(lens)
    got, w = _check(q, cache, None, kv, 0.3)
    for i, n in enumerate(lens):
        cache.k_codes[i, :, n:], cache.v_codes[i, :, n:] = 0x7f, 0xff
        for t in (cache.k_scales, cache.v_scales):
            t[i, :, -(-n // block):] = float("nan")
    w2 = torch.zeros_like(w)
    again = ops.dense_decode_fp8(q, cache, kv_len=kv, out_dtype=torch.float32, scaling=0.3, weights=w2)
    assert torch.equal(got, again) and torch.equal(w, w2)


@pytest.mark.parametrize("q_h,k_h,v_h,d", LAYOUTS)
@pytest.mark.parametrize("dtype,block", [(torch.bfloat16, 64), (torch.float16, 32)])
def test_dense_layouts_split(q_h, k_h, v_h, d, dtype, block):
    """More positions than one block of a unit takes: splits without a key, with one, and full ones are joined."""
    g = _gen(q_h * d + block + 1)
    b, L = 4, 777
    cache = F.random_cache(g, b, k_h, v_h, L, d, block)
    q = _randn(g, b, q_h, 1, d, dtype=dtype)
    got, w = _check(q, cache, None, _int32([777, 0, 129, 640]), 1 / math.sqrt(d), rows=[0, 2, 3])
    assert got[1].isnan().all() and not w[1].any()


@pytest.mark.parametrize("q_h,k_h,v_h,d,b", [(12, 1, 2, 128, 40), (15, 1, 5, 64, 30), (16, 1, 8, 64, 40)])
def test_dense_many_units(q_h, k_h, v_h, d, b):
    """Batches whose units hold several value heads (at least 128 blocks of them)."""
    g = _gen(q_h * d + b)
    cache = F.random_cache(g, b, k_h, v_h, 1500, d, 64)
    for dtype in (torch.bfloat16, torch.float16):
        q = _randn(g, b, q_h, 1, d, dtype=dtype)
        _check(q, cache, None, _int32([1500 - 37 * i for i in range(b)]), 0.1)
    m = torch.zeros(b, 1, 1, 1500, device="cuda")
    m[:, ..., 700:] = float("-inf")
    _check(q, cache, m, None, 0.1)


@pytest.mark.parametrize("q_h,k_h,v_h,d", [(12, 1, 2, 128), (15, 1, 5, 64)])
@pytest.mark.parametrize("L", [255, 257, 511, 512, 513, 8192, 8193, 16416, 70001])
def test_dense_one_row_splits(q_h, k_h, v_h, d, L):
    """One row: one block to 512 positions, 64 splits at 8192, more past it."""
    g = _gen(L + d)
    cache = F.random_cache(g, 1, k_h, v_h, L, d, 64)
    _check(_randn(g, 1, q_h, 1, d, dtype=torch.bfloat16), cache, None, None, 0.2)


@pytest.mark.parametrize("mdt", [torch.bool, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("q_h,k_h,v_h,d", [(15, 1, 5, 64), (4, 1, 2, 128)])
def test_dense_masks(mdt, per_head, q_h, k_h, v_h, d):
    g = _gen(11)
    b, L = 4, 517
    cache = F.random_cache(g, b, k_h, v_h, L, d, 32)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    shape = (b, q_h if per_head else 1, 1, L + 7)  # longer than the cache
    if mdt == torch.bool:
        m = torch.rand(shape, generator=g, device="cuda") < 0.5
    else:
        m = _randn(g, *shape)
        m[torch.rand(shape, generator=g, device="cuda") < 0.3] = float("-inf")
        m[1, ..., 5:] = torch.finfo(mdt).min
        m[2] = torch.finfo(mdt).min  # every key: the mean of the values
        m = m.to(mdt)
        m[0, ..., 100:400] = float("-inf")
    _check(q, cache, m, None, 0.125)
    _check(q, cache, m[:1, :, :, 3:], _int32([510, 3, 77, 400]), 0.125)  # off its words, one for all rows


def test_dense_empty_rows_and_nan():
    """A row without keys is NaN, as dense_decode's, and adds no weight; a NaN of a value reaches its own dim, of a key
    its row; an infinite mask its heads."""
    g = _gen(12)
    b, q_h, k_h, v_h, d, L = 5, 6, 2, 3, 64, 200
    cache = F.random_cache(g, b, k_h, v_h, L, d, 32)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    kv = _int32([0, 200, -3, 150, 170])
    mask = torch.zeros(b, 1, 1, L, device="cuda")
    mask[1] = float("-inf")
    cache.v_codes[3, 1, 20, 40] = 0x7f
    cache.k_codes[4, 0, 30, 1] = 0xff
    w = torch.ones(b, 1, L, device="cuda")
    got = ops.dense_decode_fp8(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32, weights=w)[:, :, 0]
    assert got[[0, 1, 2]].isnan().all()
    assert got[3, 2:4, 40].isnan().all() and got.isnan()[3].sum() == 2
    assert got[4, :3].isnan().all() and got[4, 3:].isfinite().all()
    assert (w[:3] == 1).all() and (w[3, :, 150:] == 1).all() and (w[4, :, 170:] == 1).all()
    assert abs(float(w[3].sum()) - L - 6) < 1e-3 and abs(float(w[4].sum()) - L - 3) < 1e-3


def test_dense_small_weights_beside_a_dominating_key():
    """One key 20 nats above the rest holds the value 0: what the many others add up to is the output."""
    g = _gen(13)
    L, d = 4096, 128
    x = torch.zeros(1, 1, L, d, device="cuda")
    x[0, 0, 7] = 1.0
    v = _randn(g, 1, 1, L, d) * 0.1 + 1.0
    v[0, 0, 7] = 0.0
    cache = ops.KVFP8(*F.quantise(x, 64), *F.quantise(v, 64), 64)
    for dtype in (torch.bfloat16, torch.float16):
        _check(torch.full((1, 1, 1, d), 20.0 / d, device="cuda").to(dtype), cache, None, None, 1.0)


def test_dense_outputs_and_weights_of_large_blocks():
    """Blocks of scales from 2^-60 to 2^60 beside each other: every one enters with its own."""
    g = _gen(14)
    L, d, block = 1024, 128, 32
    k = F.quantise(_randn(g, 1, 1, L, d), block)
    c, s = F.quantise(_randn(g, 1, 2, L, d), block)
    s = s * torch.exp2(torch.arange(32, device="cuda").float() * 4 - 60)
    cache = ops.KVFP8(*k, c, s, block)
    q = _randn(g, 1, 4, 1, d, dtype=torch.bfloat16)
    for i in (0, 13, 31):  # the mask leaves one block of each size
        m = torch.full((1, 1, 1, L), float("-inf"), device="cuda")
        m[..., 32 * i:32 * i + 32] = 0
        _check(q, cache, m, None, 0.1)


def test_weights_are_added_in_place():
    """weights_add adds below kv_len and leaves the rest; groups: any common divisor of the head counts."""
    g = _gen(15)
    b, q_h, k_h, v_h, d, L = 2, 12, 2, 4, 64, 700
    cache = F.random_cache(g, b, k_h, v_h, L, d, 64)
    kv = _int32([700, 333])
    total = torch.zeros(b, 2, L, dtype=torch.float64, device="cuda")
    w = _randn(g, b, 2, L + 5).abs()
    first = w.clone()
    for _ in range(3):
        q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
        got, one = _check(q, cache, None, kv, 0.125, G=2)
        _, both = _check(q, cache, None, kv, 0.125, G=1)
        _close(one.sum(1, keepdim=True), both.double(), 2.0 ** -20 * both.double())
        ops.dense_decode_fp8(q, cache, kv_len=kv, scaling=0.125, weights=w)
        total += one.double()
    want = first.double()
    want[..., :L] += total
    _close(w, want, 3 * U32 * want.abs())
    assert torch.equal(w[1, :, 333:], first[1, :, 333:]) and torch.equal(w[..., L:], first[..., L:])


def test_dense_expanded_batch_and_offsets_past_32_bits():
    """One cache row read by several batch rows (stride 0); a cache whose last positions lie past 2^32 bytes."""
    g = _gen(16)
    L, d, block = 1000, 64, 32
    one = F.random_cache(g, 1, 1, 1, L, d, block)
    wide = ops.KVFP8(*(t.expand(3, *t.shape[1:]) for t in one[:4]), block)
    q = _randn(g, 3, 4, 1, d, dtype=torch.bfloat16)
    got = ops.dense_decode_fp8(q, wide, kv_len=_int32([1000, 10, 500]))
    for i, n in enumerate((1000, 10, 500)):
        assert torch.equal(got[i:i + 1], ops.dense_decode_fp8(q[i:i + 1], one, kv_len=_int32([n])))
    L = (1 << 24) + 64
    big = torch.zeros(1, 1, L, 272, dtype=torch.uint8, device="cuda")[..., :d]  # 4.6 GB of rows 272 bytes apart
    far = ops.KVFP8(big, torch.ones(1, 1, L // block, device="cuda"), big, torch.ones(1, 1, L // block, device="cuda"), block)
    x = _randn(g, 64, d)
    big[0, 0, -64:] = F.nearest(x)
    m = torch.full((1, 1, 1, L), float("-inf"), dtype=torch.float16, device="cuda")
    m[..., -64:] = 0
    q = _randn(g, 1, 2, 1, d, dtype=torch.bfloat16)
    part = ops.KVFP8(big[:, :, -64:], far.k_scales[..., -2:], big[:, :, -64:], far.v_scales[..., -2:], block)
    ref, tol, _, _ = _dense_ref(q, *F.cache_values(part), None, None, 0.125)
    _close(ops.dense_decode_fp8(q, far, attention_mask=m, out_dtype=torch.float32), ref, tol + U32 * ref.abs())


# ------------------------------------------------------------------- together

def test_chain_captured_and_replayed():
    """A step (rotations, append with norms, attention with weights) in a graph on a stream of its own, the workspace
    grown in between: every replay equals the eager step at its position."""
    g = _gen(21)
    B, L, n_q, n_k, n_v, d, block = 4, 700, 12, 1, 2, 128, 32
    cache, mine = (ops.KVFP8(*(torch.zeros(s, dtype=t, device="cuda") for h in (n_k, n_v) for s, t in
                               (((B, h, L, d), torch.uint8), ((B, h, 22), torch.float32))), block) for _ in range(2))
    qkv, pos, kv = _randn(g, B, 15 * d, dtype=torch.bfloat16), _int32([0] * B), _int32([0] * B)
    table, norm = torch.empty(B, d // 2, 2, device="cuda"), (1 + 0.1 * _randn(g, d)).to(torch.bfloat16)
    q, out = torch.empty(B, n_q, d, dtype=torch.bfloat16, device="cuda"), torch.empty(B, n_q, 1, d, dtype=torch.bfloat16, device="cuda")
    w, w2 = torch.zeros(B, 1, L, device="cuda"), torch.zeros(B, 1, L, device="cuda")

    def step(c, w):
        ops.rope_table(pos, d, 1e6, out=table)
        ops.norm_rope_kv_append_fp8(qkv, n_q, table, pos, c, norm, norm, q_out=q)
        ops.dense_decode_fp8(q.view(B, n_q, 1, d), c, kv_len=kv, out=out, weights=w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, w)
    for t in (*cache[:4], *mine[:4], w, w2):
        t.zero_()
    for i in range(70):
        qkv.copy_(_randn(g, B, 15 * d) * (1 + i % 9))
        pos.fill_(i)
        kv.fill_(i + 1)
        graph.replay()
        got = out.clone()
        if i == 5:  # a larger call through the cached workspaces
            ops.dense_decode_fp8(_randn(g, 9, 12, 1, d, dtype=torch.bfloat16), F.random_cache(g, 9, 1, 2, 3000, d, 64),
                                 weights=torch.zeros(9, 1, 3000, device="cuda"))
        step(mine, w2)
        assert torch.equal(got, out), i
    assert F.same(cache, mine) and torch.equal(w, w2)
    assert abs(float(w.sum()) - B * n_q * 70) < 1.0
    ops.clear_workspaces()


def test_other_stream_and_caller_workspace():
    g = _gen(22)
    cache = F.random_cache(g, 2, 1, 2, 900, 64, 64)
    q = _randn(g, 2, 4, 1, 64, dtype=torch.float16)
    want = ops.dense_decode_fp8(q, cache)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        need = ops._lib.load().saga_dense_fp8_workspace_bytes(2, 4, 900, 64, 0)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        a, b = ops.dense_decode_fp8(q, cache), ops.dense_decode_fp8(q, cache, workspace=ws)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    with pytest.raises(ValueError, match="workspace"):
        ops.dense_decode_fp8(q, cache, workspace=ws[:256])
    with pytest.raises(RuntimeError, match="CPU fallback"):
        ops.dense_decode_fp8(q.cpu(), cache)
    with pytest.raises(RuntimeError, match="do not divide"):
        ops.dense_decode_fp8(q, cache, weights=torch.zeros(2, 2, 900, device="cuda"))
    with pytest.raises(ValueError, match="kv_len"):
        ops.dense_decode_fp8(q, cache, kv_len=_int32([1]))
    with pytest.raises(NotImplementedError):
        ops.dense_decode_fp8(_randn(g, 2, 4, 2, 64, dtype=torch.float16), cache)
