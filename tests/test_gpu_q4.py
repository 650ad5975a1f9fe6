"""Operators on data held in 4 bits (weights, key / value cache) on the GPU against 64-bit arithmetic."""
import math

import pytest
import torch

import q4_util as Q
from saga_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def _close(got, ref, tol):
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(((got.double() - ref).abs() / tol).max()))
    assert torch.isfinite(got).all()


# ------------------------------------------------------------------- weights

def _gemv_ref(x, w, rms):
    """x w^T in 64 bits and, per output, a bound of the kernel's fp32 error: at most K / 16 + 64 roundings, each of
    half a step of a partial sum of x (s (16 + c)) and x (z - 16 s)."""
    W = Q.weight_values(w)
    s, z = (t.transpose(1, 2).reshape(W.shape[0], -1).repeat_interleave(w.group, 1).double()
            for t in (w.scales[..., 0], w.scales[..., 1]))
    xd = x.double()
    size = xd.abs() @ (31 * s + (z - 16 * s).abs()).t() * (x.shape[1] / 16 + 64) * U32
    y = xd @ W.t()
    if rms is not None:
        r = 1 / (xd.square().mean(-1, keepdim=True) + rms).sqrt()
        y, size = y * r, size * r + (y * r).abs() * (x.shape[1] / 16 + 64) * U32
    return y, size


SHAPES = [(1, 16, 32, 32), (8, 1536, 1536, 64), (5, 64, 960, 64), (16, 1920, 1536, 128), (17, 960, 2560, 32), (32, 48, 128, 128),
          (3, 1536, 8960, 64), (32, 4096, 96, 32), (2, 8192, 256, 64), (9, 32, 12416, 64), (1, 151936, 128, 128),
          (32, 17920, 192, 64), (20, 64, 8960, 128), (7, 112, 1600, 64), (9, 65552, 320, 64), (32, 65568, 960, 32),
          (18, 65552, 1536, 32), (2, 65536, 2048, 128), (31, 65552, 2944, 64),
          (6, 4096, 1536, 64), (25, 4112, 512, 128), (16, 5120, 960, 32), (24, 12304, 1600, 64), (1, 32768, 3200, 128)]


@pytest.mark.parametrize("M,N,K,group", SHAPES)
@pytest.mark.parametrize("rms", [None, 1e-5])
def test_gemv_q4_store_and_bias(M, N, K, group, rms):
    g = _gen(M * K + N)
    x = _randn(g, M, K, dtype=torch.bfloat16)
    w = ops.quantize_gemv_weight(0.05 * _randn(g, N, K) + 0.02, group)
    bias = _randn(g, N, dtype=torch.bfloat16)
    ref, size = _gemv_ref(x, w, rms)
    got = ops.gemv_q4(x, w, rms_eps=rms)
    _close(got, ref, HALF[torch.bfloat16] * (ref.abs() + size) + size)
    ref = ref + bias.double()
    _close(ops.gemv_q4(x, w, bias=bias, rms_eps=rms), ref, HALF[torch.bfloat16] * (ref.abs() + size) + size + U32 * ref.abs())
    again = ops.gemv_q4(x, w, rms_eps=rms)
    assert torch.equal(got, again)  # no order that changes


@pytest.mark.parametrize("M,N,K,group", SHAPES[:8] + SHAPES[-10:])
def test_gemv_q4_add_and_silu(M, N, K, group):
    g = _gen(N + K)
    xs = _randn(g, M, K + 8, dtype=torch.bfloat16)
    x = xs[:, :K]  # rows with a stride of their own
    w = ops.quantize_gemv_weight(0.05 * _randn(g, N, K), group)
    ref, size = _gemv_ref(x, w, None)
    wide = _randn(g, M, N + 3, dtype=torch.bfloat16)
    out = wide[:, :N]
    want = out.double() + ref
    rest = wide[:, N:].clone()
    ops.gemv_q4(x, w, epilogue="add", out=out)
    _close(out, want, HALF[torch.bfloat16] * (want.abs() + size) + size + U32 * want.abs())
    assert torch.equal(wide[:, N:], rest)
    ref, size = _gemv_ref(x, w, 1e-6)
    gate, up, eg, eu = ref[:, 0::2], ref[:, 1::2], size[:, 0::2], size[:, 1::2]
    want = gate * torch.sigmoid(gate) * up
    # |silu'| <= 1.1, |silu(g)| <= |g|; the activation itself: 8 roundings
    tol = 1.1 * eg * (up.abs() + eu) + gate.abs() * eu + 8 * U32 * want.abs()
    _close(ops.gemv_q4(x, w, rms_eps=1e-6, epilogue="silu_pairs"), want, HALF[torch.bfloat16] * (want.abs() + tol) + tol)


@pytest.mark.parametrize("M,N,K", [(32, 4144, 1824), (19, 4112, 1280), (17, 4096, 1536), (24, 8208, 480), (31, 4112, 2048)])
def test_gemv_q4_streamed_32_rows(M, N, K):
    """Groups of 32 under 17 to 32 rows: sums of x as operands; NaN stays in its row of x and its row of W."""
    g = _gen(N + K + 1)
    x = _randn(g, M, K, dtype=torch.bfloat16)
    w = ops.quantize_gemv_weight(0.05 * _randn(g, N, K) + 0.02, 32)
    ref, size = _gemv_ref(x, w, 1e-6)
    got = ops.gemv_q4(x, w, rms_eps=1e-6)
    _close(got, ref, HALF[torch.bfloat16] * (ref.abs() + size) + size)
    w.scales[N // 16 - 1, K // 32 - 1, 5] = float("nan")
    x[M - 1, 3] = float("nan")
    bad = ops.gemv_q4(x, w, rms_eps=1e-6)
    n = N - 16 + 5
    assert bad[:, n].isnan().all() and bad[M - 1].isnan().all()
    keep = torch.arange(N, device="cuda") != n
    assert torch.equal(bad[: M - 1][:, keep], got[: M - 1][:, keep])


def test_gemv_q4_special_values():
    """Rows of x do not meet each other; constant, tiny and one-sided groups; a NaN offset reaches its own row."""
    g = _gen(3)
    W = _randn(g, 32, 256)
    W[0] = 0
    W[1] = 0.75
    W[2] = 1e-7 * _randn(g, 256)
    W[3] = 100 + 0.01 * _randn(g, 256)
    W[4, ::2] = -60000.0
    w = ops.quantize_gemv_weight(W, 64)
    assert ((Q.weight_values(w) - W.double()).abs() <= 0.500001 * w.scales[..., 0].transpose(1, 2).reshape(32, 4)
            .repeat_interleave(64, 1).double()).all()
    x = _randn(g, 6, 256, dtype=torch.bfloat16)
    ref, size = _gemv_ref(x, w, None)
    _close(ops.gemv_q4(x, w), ref, HALF[torch.bfloat16] * (ref.abs() + size) + size)
    x[2, 5], x[4, 7] = float("inf"), float("nan")
    got = ops.gemv_q4(x, w)
    keep = [0, 1, 3, 5]
    _close(got[keep], ref[keep], (HALF[torch.bfloat16] * (ref.abs() + size) + size)[keep])
    assert got[4].isnan().all() and not got[2].isfinite().any()
    w.scales[1, 2, 5, 1] = float("nan")
    got = ops.gemv_q4(x[keep], w)
    assert got[:, 21].isnan().all() and got.isnan().sum() == 4


@pytest.mark.parametrize("N,K,group", [(16, 32, 32), (1920, 1536, 64), (960, 960, 32), (64, 8960, 128), (48, 192, 64)])
def test_unpack_gemv_q4(N, K, group):
    g = _gen(N + K)
    w = ops.quantize_gemv_weight(_randn(g, N, K), group)
    v = ops.quantize_gemv_weight(_randn(g, 64, 256), 64)
    ref = Q.weight_values(w).float().to(torch.bfloat16)  # one sum of 15 exact bits and z: one rounding to fp32
    a, b, c = ops.unpack_gemv_q4([w, v, w], [None, (2, 16), (1, N)])
    assert torch.equal(a, ref)
    vr = Q.weight_values(v).float().to(torch.bfloat16)
    order = torch.cat([h * 16 + torch.cat([torch.arange(0, 16, 2), torch.arange(1, 16, 2)]) for h in range(2)])
    assert torch.equal(b, torch.cat([vr[order.cuda()], vr[32:]]))
    assert torch.equal(c, torch.cat([ref[0::2], ref[1::2]]))


# ------------------------------------------------------------------- cache rows

def _tokens(g, n, n_q, n_k, n_v, d, dtype):
    x = _randn(g, n, (n_q + n_k + n_v) * d)
    x.view(n, -1, d)[:, :, ::7] += 3.0  # offsets, as biased projections have
    return x.to(dtype)


def _rotate(qkv, table, n_q, n_k, d, dtype):
    x = qkv.to(dtype).reshape(qkv.shape[0], -1, d)
    cs, sn = table[:, None, :, 0].to(dtype), table[:, None, :, 1].to(dtype)
    x1, x2 = x[:, : n_q + n_k, : d // 2], x[:, : n_q + n_k, d // 2:]
    return torch.cat([x1 * cs - x2 * sn, x2 * cs + x1 * sn], -1), x[:, n_q + n_k:]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_q,n_k,n_v,d,group", [(12, 1, 2, 128, 64), (15, 1, 5, 64, 32), (4, 2, 2, 128, 32), (5, 5, 1, 64, 64)])
@pytest.mark.parametrize("n", [1, 7, 333])
def test_append_and_read(n, n_q, n_k, n_v, d, group, dtype):
    """Codes, scales and offsets equal the rule's in fp32 (the same operations: IEEE additions, products and quotients),
    every value is within s / 2 of the 64-bit one, other rows stay as they were, reading back gives s c + z."""
    g = _gen(n + d + n_q)
    B, L = 3, 400
    qkv = _tokens(g, n, n_q, n_k, n_v, d, dtype)
    pos = torch.randperm(L, generator=g, device="cuda")[:n].int()
    batch = torch.randint(0, B, (n,), generator=g, device="cuda").int()
    table = ops.rope_table(pos, d, 1e4)
    cache = Q.random_cache(g, B, n_k, n_v, L, d, group)
    before = [t.clone() for t in cache]
    q = ops.rope_kv_append_q4(qkv, n_q, table, pos, cache, batch=batch)
    rot, v = _rotate(qkv, table, n_q, n_k, d, torch.float32)
    assert torch.equal(q, rot[:, :n_q].to(dtype))
    want = [t.clone() for t in before]
    for x, kind, at in ((rot[:, n_q:], "k", 0), (v, "v", 2)):
        codes, sz = Q.quantise(x.cpu(), group)
        want[at][batch.long(), :, pos.long()] = Q.pack_row(codes, kind).cuda()
        want[at + 1][batch.long(), :, pos.long()] = sz.cuda()
    for a, b in zip(cache, want):
        assert torch.equal(a, b)
    rot64, v64 = _rotate(qkv, table, n_q, n_k, d, torch.float64)
    kf, vf = ops.read_kv_q4(cache, pos, batch, dtype=torch.float32)
    for x, got, sz in ((rot64[:, n_q:], kf, cache.k_scales), (v64, vf, cache.v_scales)):
        s = sz[batch.long(), :, pos.long()].double()[..., 0::2].repeat_interleave(group, -1)
        assert ((got.double() - x).abs() <= s * (0.5 + 2 ** -18) + 2 ** -20 * x.abs().amax()).all()
    for name, got in zip(("k", "v"), ops.read_kv_q4(cache, pos, batch, dtype=dtype)):
        held = Q.values(Q.open_row(getattr(cache, name + "_codes")[batch.long(), :, pos.long()], name),
                        getattr(cache, name + "_scales")[batch.long(), :, pos.long()], torch.float32)
        assert torch.equal(got, held.to(dtype))


def test_append_out_of_range_and_special_values():
    """Indices out of range write nothing and give NaN queries and reads; NaN, infinite and too large groups read back
    as NaN beside groups that do not; constant, zero and tiny groups; far positions' rows only."""
    g, d = _gen(5), 64
    B, L, n_q, n_k, n_v = 2, 40, 2, 1, 1
    qkv = _tokens(g, 6, n_q, n_k, n_v, d, torch.float32)
    v = qkv.view(6, 4, d)[:, 3]
    v[0, 3], v[1, 40], v[2, 0] = float("nan"), float("-inf"), 65600.0
    v[0, 32:] = 0.0
    v[1, :32] = 1.0 / 3
    v[2, 32:] = 1e-9 * torch.arange(32, device="cuda")
    v[5, :32] = -65504.0
    v[5, 32:48] = 65504.0
    pos = torch.tensor([0, 39, 7, -1, 40, 8], dtype=torch.int32, device="cuda")
    batch = torch.tensor([0, 1, 0, 1, 0, 1], dtype=torch.int32, device="cuda")
    table = ops.rope_table(pos, d, 1e4)
    cache = Q.random_cache(g, B, n_k, n_v, L, d, 32)
    before = [t.clone() for t in cache]
    q = ops.rope_kv_append_q4(qkv, n_q, table, pos, cache, batch=batch)
    assert q[[3, 4]].isnan().all() and q[[0, 1, 2, 5]].isfinite().all()
    at = [[0, 1, 0, 1], [0, 39, 7, 8]]
    for t, b in zip(cache, before):
        b[at[0], :, at[1]] = t[at[0], :, at[1]]
        assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
    k, got = ops.read_kv_q4(cache, pos, batch, dtype=torch.float32)
    assert k[[3, 4]].isnan().all() and got[[3, 4]].isnan().all()
    got = got[:, 0]
    assert got[0, :32].isnan().all() and got[1, 32:].isnan().all() and got[2, :32].isnan().all()
    assert (got[0, 32:] == 0).all() and (got[1, :32] - 1.0 / 3).abs().max() <= 2.0 ** -15  # steps of 2^-11 / 15 .. 2^-12
    assert got[2, 32:].abs().max() <= 2.0 ** -24 and (got[5, :32] == -65504).all()
    assert (got[5, 32:48] - 65504).abs().max() <= (65504 - v[5, 48:].min()) / 30 * 1.01
    ops.rope_kv_append_q4(qkv[:2], n_q, table[:2].contiguous(), pos[[5, 5]].contiguous(), cache)  # rows 0 and 1 without batch
    with pytest.raises(RuntimeError, match="without batch"):
        ops.rope_kv_append_q4(qkv[:3], n_q, table[:3].contiguous(), pos[:3].contiguous(), cache)


def test_append_strided_and_unaligned():
    """Views: a projection row offset, caches with gaps between positions and heads."""
    g, d = _gen(6), 128
    B, L, n_q, n_k, n_v, n, group = 2, 64, 4, 1, 2, 9, 64
    big = _tokens(g, n, n_q, n_k, n_v, d, torch.bfloat16)
    wide = torch.zeros(n, big.shape[1] + 9, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:-8] = big
    pos = torch.randperm(L, generator=g, device="cuda")[:n].int()
    batch = (torch.arange(n, device="cuda") % B).int()
    table = ops.rope_table(pos, d, 1e4)
    plain = ops.KVQ4(*(torch.zeros_like(t) for t in Q.random_cache(g, B, n_k, n_v, L, d, group)))
    gaps = ops.KVQ4(*(torch.zeros(B, L, 3, 2 * t.shape[-1], dtype=t.dtype, device="cuda").transpose(1, 2)[:, : t.shape[1], :, : t.shape[-1]]
                      for t in plain))
    q = ops.rope_kv_append_q4(big, n_q, table, pos, plain, batch=batch)
    q2 = ops.rope_kv_append_q4(wide[:, 1:-8], n_q, table, pos, gaps, batch=batch)
    assert torch.equal(q, q2) and all(torch.equal(a, b) for a, b in zip(plain, gaps))
    assert all(torch.equal(a, b) for a, b in zip(ops.read_kv_q4(plain, pos, batch), ops.read_kv_q4(gaps, pos, batch)))
    query = _randn(g, B, n_q, 1, d, dtype=torch.bfloat16)
    kv = torch.tensor([L, L // 2], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.dense_decode_q4(query, plain, kv_len=kv), ops.dense_decode_q4(query, gaps, kv_len=kv))


# ------------------------------------------------------------------- attention

def _dense_ref(q, cache, mask, kv_len, scale):
    """Attention in 64 bits and, per output, a bound of the kernel's error before its last rounding:
    a score's fp32 sums (at most 64 roundings of its largest partial sum, and the mask's) move each weight by twice that
    relative, the exponential by 2^-20; a weight's terms keep 16 bits (2^-17 of s c), sums over the positions at most
    L / 16 + 64 roundings of partial sums of p s (16 + c) and p z."""
    b, q_h, _, d = q.shape
    k, v = Q.cache_values(cache)
    kz, vz = (t.unflatten(-1, (-1, 2)).double() for t in (cache.k_scales, cache.v_scales))
    group = d // kz.shape[-2]
    L = k.shape[2]
    out, tol = (torch.empty(b, q_h, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        n = L if kv_len is None else min(int(kv_len[i]), L)
        for h in range(q_h):
            kh, vh = h * k.shape[1] // q_h, h * v.shape[1] // q_h
            qd = q[i, h, 0].double()
            x = k[i, kh, :n] @ qd * scale
            qa = qd.abs().reshape(-1, group).sum(-1)
            e = ((31 * kz[i, kh, :n, :, 0] + (kz[i, kh, :n, :, 1] - 16 * kz[i, kh, :n, :, 0]).abs()) @ qa) * scale * 64 * U32
            if mask is not None:
                m = mask[i % mask.shape[0], h % mask.shape[1], 0, :n].double()
                x = x + m
                e = e + torch.where(m.isfinite(), m.abs().clamp(max=1e6), torch.zeros_like(m)) * U32
            p = torch.softmax(x, 0)
            out[i, h] = p @ v[i, vh, :n]
            ew = (2 * float(e.max()) + 2.0 ** -20) if n else 0.0
            ps = (p @ vz[i, vh, :n, :, 0]).repeat_interleave(group)
            pz = (p @ vz[i, vh, :n, :, 1].abs()).repeat_interleave(group)
            tol[i, h] = (2 * ew * (p @ v[i, vh, :n].abs() + out[i, h].abs()) + 2.0 ** -17 * 15 * ps
                         + (n / 16 + 64) * U32 * (31 * ps + pz))
    return out[:, :, None], tol[:, :, None]


LAYOUTS = [(12, 1, 2, 128), (12, 2, 2, 128), (15, 1, 5, 64), (15, 5, 5, 64), (12, 3, 2, 64), (12, 4, 1, 128), (32, 1, 2, 64),
           (6, 6, 6, 128), (16, 1, 1, 64), (24, 1, 8, 128), (1, 1, 1, 64), (12, 2, 3, 128), (40, 2, 1, 64)]


@pytest.mark.parametrize("q_h,k_h,v_h,d", LAYOUTS)
@pytest.mark.parametrize("dtype,group", [(torch.bfloat16, 64), (torch.bfloat16, 32), (torch.float16, 64), (torch.float16, 32)])
def test_dense_q4_layouts(q_h, k_h, v_h, d, dtype, group):
    g = _gen(q_h * d + group)
    b, L = 3, 301
    cache = Q.random_cache(g, b, k_h, v_h, L, d, group)
    q = _randn(g, b, q_h, 1, d, dtype=dtype)
    kv = torch.tensor([301, 1, 133], dtype=torch.int32, device="cuda")
    ref, tol = _dense_ref(q, cache, None, kv, 1 / math.sqrt(d))
    _close(ops.dense_decode_q4(q, cache, kv_len=kv, out_dtype=torch.float32), ref, tol + U32 * ref.abs())
    _close(ops.dense_decode_q4(q, cache, kv_len=kv), ref, tol + HALF[dtype] * (ref.abs() + tol))


@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 1000, 4099, 33000])
@pytest.mark.parametrize("b", [1, 9])
def test_dense_q4_lengths(L, b):
    """Lengths around the steps, splits and blocks; what lies behind kv_len holds NaN scales."""
    g = _gen(L + b)
    q_h, k_h, v_h, d, group = 12, 1, 2, 128, 64
    cache = Q.random_cache(g, b, k_h, v_h, L, d, group)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    lens = [max(1, L - (3 * L // 4) * i // b) for i in range(b)]
    for i, n in enumerate(lens):
        for t in (cache.k_scales, cache.v_scales):
            t[i, :, n:] = float("nan")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ref, tol = _dense_ref(q, cache, None, kv, 0.3)
    got = ops.dense_decode_q4(q, cache, kv_len=kv, out_dtype=torch.float32, scaling=0.3)
    _close(got, ref, tol + U32 * ref.abs())
    assert torch.equal(got, ops.dense_decode_q4(q, cache, kv_len=kv, out_dtype=torch.float32, scaling=0.3))


@pytest.mark.parametrize("q_h,k_h,v_h,d", LAYOUTS)
@pytest.mark.parametrize("dtype,group", [(torch.bfloat16, 64), (torch.bfloat16, 32), (torch.float16, 64)])
def test_dense_q4_layouts_split(q_h, k_h, v_h, d, dtype, group):
    """More positions than one block of a unit takes: splits without a key, with one, and full ones are joined."""
    g = _gen(q_h * d + group + 1)
    b, L = 4, 777
    cache = Q.random_cache(g, b, k_h, v_h, L, d, group)
    q = _randn(g, b, q_h, 1, d, dtype=dtype)
    kv = torch.tensor([777, 0, 129, 640], dtype=torch.int32, device="cuda")
    ref, tol = _dense_ref(q, cache, None, kv, 1 / math.sqrt(d))
    got = ops.dense_decode_q4(q, cache, kv_len=kv, out_dtype=torch.float32)
    assert got[1].isnan().all()
    keep = [0, 2, 3]
    _close(got[keep], ref[keep], tol[keep] + U32 * ref[keep].abs())


@pytest.mark.parametrize("q_h,k_h,v_h,d", [(12, 1, 2, 128), (15, 1, 5, 64)])
@pytest.mark.parametrize("L", [255, 257, 511, 512, 513, 8192, 8193, 16416, 70001])
def test_dense_q4_one_row_splits(q_h, k_h, v_h, d, L):
    """One row: one block to 512 positions, 64 splits at 8192, 65 (joined by blocks of 32 dims) and more past it."""
    g = _gen(L + d)
    cache = Q.random_cache(g, 1, k_h, v_h, L, d, 64)
    q = _randn(g, 1, q_h, 1, d, dtype=torch.bfloat16)
    ref, tol = _dense_ref(q, cache, None, None, 0.2)
    got = ops.dense_decode_q4(q, cache, out_dtype=torch.float32, scaling=0.2)
    _close(got, ref, tol + U32 * ref.abs())


@pytest.mark.parametrize("mdt", [torch.bool, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_head", [False, True])
def test_dense_q4_masks(mdt, per_head):
    g = _gen(11)
    b, q_h, k_h, v_h, d, L = 4, 15, 1, 5, 64, 517
    cache = Q.random_cache(g, b, k_h, v_h, L, d, 32)
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
    ref, tol = _dense_ref(q, cache, m[..., :L].to(torch.float32) if mdt == torch.bool else m[..., :L], None, 0.125)
    _close(ops.dense_decode_q4(q, cache, attention_mask=m, out_dtype=torch.float32), ref, tol + U32 * ref.abs())


def test_dense_q4_empty_rows_and_nan():
    """A row without keys is NaN, as dense_decode's; a NaN group of a value reaches its own dims, of a key its row."""
    g = _gen(12)
    b, q_h, k_h, v_h, d, L = 5, 6, 2, 3, 64, 200
    cache = Q.random_cache(g, b, k_h, v_h, L, d, 32)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    kv = torch.tensor([0, 200, -3, 150, 170], dtype=torch.int32, device="cuda")
    mask = torch.zeros(b, 1, 1, L, device="cuda")
    mask[1] = float("-inf")
    cache.v_scales[3, 1, 20, 2] = float("nan")
    cache.k_scales[4, 0, 30, 1] = float("nan")
    got = ops.dense_decode_q4(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32)[:, :, 0]
    assert got[[0, 1, 2]].isnan().all()
    assert got[3, 2:4, 32:].isnan().all() and got[3, :, :32].isfinite().all() and got[3, [0, 1, 4, 5]].isfinite().all()
    assert got[4, :3].isnan().all() and got[4, 3:].isfinite().all()


def test_dense_q4_small_weights_beside_a_dominating_key():
    """One key 20 nats above the rest holds the value 0: what the many others add up to is the output."""
    g = _gen(13)
    b, L, d = 1, 4096, 128
    x = torch.zeros(1, 1, L, d, device="cuda")
    x[0, 0, 7] = 1.0
    v = _randn(g, 1, 1, L, d) * 0.1 + 1.0
    v[0, 0, 7] = 0.0
    parts = []
    for t, kind in ((x, "k"), (v, "v")):
        c, sz = Q.quantise(t, 64)
        parts += [Q.pack_row(c, kind), sz]
    cache = ops.KVQ4(*parts)
    for dtype in (torch.bfloat16, torch.float16):
        q = torch.full((1, 1, 1, d), 20.0 / d, device="cuda").to(dtype)
        ref, tol = _dense_ref(q, cache, None, None, 1.0)
        assert float(tol.max() / ref.abs().min()) < 1e-3
        _close(ops.dense_decode_q4(q, cache, scaling=1.0, out_dtype=torch.float32), ref, tol + U32 * ref.abs())


# ------------------------------------------------------------------- together

def test_chain_captured_and_replayed():
    """A layer's step as a decoder runs it (projection, append, attention, output projection into the residual stream)
    captured in a graph on a stream of its own: every replay equals the eager step at its position."""
    g = _gen(21)
    B, L, n_q, n_k, n_v, d, H = 4, 96, 12, 1, 2, 128, 256
    w_in = ops.quantize_gemv_weight(0.1 * _randn(g, (n_q + n_k + n_v) * d, H), 64)
    w_out = ops.quantize_gemv_weight(0.1 * _randn(g, H, n_q * d), 128)
    start = Q.random_cache(g, B, n_k, n_v, L, d, 64)
    x0 = _randn(g, B, H, dtype=torch.bfloat16)

    def state():
        return (x0.clone(), torch.full((B,), 40, dtype=torch.int32, device="cuda"),
                torch.full((B,), 41, dtype=torch.int32, device="cuda"), ops.KVQ4(*(t.clone() for t in start)))

    def step(x, pos, kv, cache):
        qkv = ops.gemv_q4(x, w_in, rms_eps=1e-6)
        q = ops.rope_kv_append_q4(qkv, n_q, ops.rope_table(pos, d, 1e4), pos, cache)
        a = ops.dense_decode_q4(q.view(B, n_q, 1, d), cache, kv_len=kv)
        ops.gemv_q4(a.view(B, n_q * d), w_out, epilogue="add", out=x)
        ops.advance_positions(pos, kv)

    eager, held = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*held)
    for _ in range(5):
        graph.replay()
        step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1])
        assert all(torch.equal(a, b) for a, b in zip(held[3], eager[3]))
    q, v = ops.read_kv_q4(held[3], held[1] - 1)
    assert q.isfinite().all() and v.isfinite().all()


# ------------------------------------------------------------------- large offsets, workspaces, streams

@pytest.mark.parametrize("kind", ["batch", "position"])
def test_cache_offsets_past_32_bits(kind):
    """Caches whose batch rows, or whose positions, lie more than 4 GB apart: the same results as compact ones."""
    g = _gen(31)
    b, L = (2, 40) if kind == "batch" else (1, 75)
    q_h, k_h, v_h, d = 12, 1, 2, 128
    compact = Q.random_cache(g, b, k_h, v_h, L, d, 64)
    big = torch.empty((1 << 32) + (1 << 30), dtype=torch.uint8, device="cuda")
    halves = torch.empty((1 << 31) + (1 << 29), dtype=torch.float16, device="cuda")

    def spread(t, base, off):
        n, row = t.shape[1], t.shape[-1]
        if kind == "batch":
            strides = ((1 << 32) // base.element_size() + 4096, L * row, row, 1)
        else:
            strides = (16, row, 60_000_000 // base.element_size(), 1)
        return base.as_strided(t.shape, strides, off)

    far = ops.KVQ4(spread(compact[0], big, 0), spread(compact[1], halves, 0), spread(compact[2], big, 65536),
                   spread(compact[3], halves, 65536))
    for t, c in zip(far, compact):
        t.copy_(c)
    q = _randn(g, b, q_h, 1, d, dtype=torch.bfloat16)
    assert torch.equal(ops.dense_decode_q4(q, far), ops.dense_decode_q4(q, compact))
    pos = torch.full((b,), L - 1, dtype=torch.int32, device="cuda")
    qkv = _tokens(g, b, q_h, k_h, v_h, d, torch.bfloat16)
    table = ops.rope_table(pos, d, 1e4)
    for cache in (far, compact):
        ops.rope_kv_append_q4(qkv, q_h, table, pos, cache)
    assert all(torch.equal(t, c) for t, c in zip(far, compact))
    assert all(torch.equal(x, y) for x, y in zip(ops.read_kv_q4(far, pos), ops.read_kv_q4(compact, pos)))


@pytest.mark.parametrize("N,K", [(1 << 20, 8704), ((1 << 23) + 512, 1024)])
def test_weight_offsets_past_32_bits(N, K):
    """Codes of more than 4 GB: the first and the last rows against 64 bits."""
    g = _gen(32)
    codes = torch.empty(N // 16, (K + 127) // 128, 1024, dtype=torch.uint8, device="cuda").random_(0, 256, generator=g)
    scales = torch.empty(N // 16, K // 128, 16, 2, dtype=torch.float16, device="cuda").uniform_(0.01, 0.02, generator=g)
    w = ops.Q4Weight(codes, scales, 128)
    x = _randn(g, 3, K, dtype=torch.bfloat16)
    got = ops.gemv_q4(x, w)
    for part in (slice(0, 4), slice(N // 16 - 4, N // 16)):
        ref, size = _gemv_ref(x, ops.Q4Weight(codes[part], scales[part], 128), None)
        rows = slice(16 * part.start, 16 * part.stop)
        _close(got[:, rows], ref, HALF[torch.bfloat16] * (ref.abs() + size) + size)
    assert got.isfinite().all()


def test_gemv_q4_workspaces():
    """Split over K or not, in the cached workspace or the caller's: within the bound of each; a workspace of another
    type, size or device is refused."""
    g = _gen(33)
    x = _randn(g, 8, 8960, dtype=torch.bfloat16)
    w = ops.quantize_gemv_weight(0.05 * _randn(g, 256, 8960), 64)
    need = ops._lib.load().saga_gemv_q4_workspace_bytes(8, 256, 8960)
    assert need > 0
    ref, size = _gemv_ref(x, w, 1e-6)
    own = torch.empty(need, dtype=torch.uint8, device="cuda")
    a, b, c = (ops.gemv_q4(x, w, rms_eps=1e-6, **kw) for kw in ({}, {"workspace": own}, {"split_k": False}))
    assert torch.equal(a, b)
    for got in (a, c):
        _close(got, ref, HALF[torch.bfloat16] * (ref.abs() + size) + size)
    for bad in (own[:-1], own.view(torch.int8), torch.empty(need)):
        with pytest.raises(ValueError, match="workspace"):
            ops.gemv_q4(x, w, workspace=bad)


def test_python_refusals():
    g = _gen(34)
    cache = Q.random_cache(g, 2, 1, 1, 8, 64, 32)
    w = ops.quantize_gemv_weight(torch.zeros(16, 128, device="cuda"), 64)
    x = torch.zeros(2, 192, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="does not meet"):
        ops.gemv_q4(x, w)
    with pytest.raises(ValueError, match="needs out"):
        ops.gemv_q4(x[:, :128].contiguous(), w, epilogue="add")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    table = ops.rope_table(pos, 64, 1e4)
    for kw, needle in ((dict(pos=pos.long()), "pos"), (dict(pos=pos[:1]), "pos"), (dict(batch=pos.long()), "batch"),
                       (dict(rope_table=table[:1]), "rope_table"), (dict(rope_table=table.double()), "rope_table")):
        a = dict(rope_table=table, pos=pos, batch=pos)
        a.update(kw)
        with pytest.raises(ValueError, match=needle):
            ops.rope_kv_append_q4(x, 1, cache=cache, **a)
    q = torch.zeros(2, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="kv_len"):
        ops.dense_decode_q4(q, cache, kv_len=pos[:1])
    with pytest.raises(ValueError, match="kv_len"):
        ops.dense_decode_q4(q, cache, kv_len=pos.long())
    with pytest.raises(NotImplementedError, match="l_q"):
        ops.dense_decode_q4(q.expand(2, 1, 2, 64), cache)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.dense_decode_q4(q, cache._replace(k_codes=cache.k_codes.cpu()))


def test_another_stream():
    """Calls on a stream of their own, each with the workspace of that stream, beside calls on the default one."""
    g = _gen(35)
    cache = Q.random_cache(g, 2, 1, 2, 3000, 128, 64)
    qs = [_randn(g, 2, 12, 1, 128, dtype=torch.bfloat16) for _ in range(2)]
    want = [ops.dense_decode_q4(q, cache) for q in qs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [[], []]
    for _ in range(8):
        got[0].append(ops.dense_decode_q4(qs[0], cache))
        with torch.cuda.stream(side):
            got[1].append(ops.dense_decode_q4(qs[1], cache))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
