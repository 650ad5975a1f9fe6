"""The forms of the 4-bit kernels that sizes choose, on the GPU: projections split over K with every epilogue, units of
several value heads in attention, masks of the type's lowest value, weights opened four units a block, appends of many
tokens in several passes, and a decoder's cache against keys and values in 64 bits.

Where the data allow it the comparison is exact: with small whole numbers and powers of two as scales every product and
partial sum of the kernels is a multiple of one unit below 2^24 of it, which fp32 holds in any order."""
import math

import pytest
import torch

import q4_util as Q
from saga_amd import ops
from saga_amd.decoder import SagaDecoder
from test_gpu_q4 import HALF, U32, _close, _gen, _randn, _rotate, _tokens
from test_gpu_q4_decoder import SHAPES, _held, _weights64

pytestmark = pytest.mark.gpu


def _ints(g, lo, hi, *size):
    return torch.randint(lo, hi + 1, size, generator=g, device="cuda")


# ------------------------------------------------------------------- weights

def _whole_weight(g, N, K, group):
    """Random codes, scales 2^-3 .. 2^-5, offsets of at most 16 / 32: multiples of 2^-5, at most 60 / 32 + 1/2."""
    codes = _ints(g, 0, 255, N // 16, (K + 127) // 128, 1024).to(torch.uint8)
    s = 2.0 ** -_ints(g, 3, 5, N // 16, K // group, 16)
    z = _ints(g, -16, 16, N // 16, K // group, 16) / 32
    return ops.Q4Weight(codes, torch.stack([s, z], -1).half(), group)


# split over K: 8 rows of x or more, 24 units of 128 columns or more; an odd number of 16-row tiles takes them one by
# one, and K % 128 != 0 ends in half a unit
SPLIT = [(8, 1536, 8960, 64), (32, 1536, 8960, 32), (16, 960, 8960, 128), (9, 48, 3200, 64), (25, 16, 8960, 32),
         (17, 2032, 3232, 32), (8, 1552, 5024, 32)]
WHOLE = [(1, 1536, 1536, 64), (7, 1536, 8960, 64), (20, 112, 1600, 32), (5, 17920, 1536, 128), (32, 8192, 3200, 64)]


@pytest.mark.parametrize("M,N,K,group", SPLIT + WHOLE)
@pytest.mark.parametrize("split_k", [True, False])
def test_gemv_q4_is_exact_on_whole_numbers(M, N, K, group, split_k):
    """x of -2 .. 2: sums of x (b + c) and of x b stay below K * 2 * 143 * 4 = 10.3 M units of 2^-5."""
    need = ops._lib.load().saga_gemv_q4_workspace_bytes(M, N, K)
    assert (need > 0) == ((M, N, K, group) in SPLIT)
    g = _gen(M + N + K)
    w = _whole_weight(g, N, K, group)
    x = _ints(g, -2, 2, M, K).to(torch.bfloat16)
    y = x.double() @ Q.weight_values(w).t()
    assert torch.equal(ops.gemv_q4(x, w, split_k=split_k), y.to(torch.bfloat16))
    bias = _ints(g, -128, 128, N).to(torch.bfloat16)
    assert torch.equal(ops.gemv_q4(x, w, bias=bias, split_k=split_k), (y + bias.double()).to(torch.bfloat16))
    wide = _ints(g, -256, 256, M + 1, N + 5).to(torch.bfloat16)  # rows with a stride of their own, and one behind the last
    held, out = wide.clone(), wide[:M, :N]
    ops.gemv_q4(x, w, epilogue="add", out=out, split_k=split_k)
    assert torch.equal(out, (held[:M, :N].double() + y).to(torch.bfloat16))
    held[:M, :N] = out
    assert torch.equal(wide, held)
    # the norm's factor: a quotient, a sum, a reciprocal root of at most 2 units and a product, 2^-21 in all; the
    # activation 8 roundings; |silu'| <= 1.1
    y = y / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    gate, up = y[:, 0::2], y[:, 1::2]
    want = gate * torch.sigmoid(gate) * up
    tol = 2.0 ** -21 * (1.1 * (gate * up).abs() + want.abs()) + 8 * U32 * want.abs()
    _close(ops.gemv_q4(x, w, rms_eps=1e-6, epilogue="silu_pairs", split_k=split_k), want,
           HALF[torch.bfloat16] * (want.abs() + tol) + tol)


@pytest.mark.parametrize("N,K,group", [(8192, 1600, 64), (5136, 8960, 128), (17920, 672, 32)])
def test_unpack_gemv_q4_four_units_a_block(N, K, group):
    """Weights of 1024 blocks of four units or more, the last block of a row of tiles not full."""
    assert N // 16 * ((K + 511) // 512) >= 1024 and (K + 127) // 128 % 4
    g = _gen(N + K)
    w = ops.quantize_gemv_weight(_randn(g, N, K), group)
    small = ops.quantize_gemv_weight(_randn(g, 32, 96), 32)
    ref = Q.weight_values(w).float().to(torch.bfloat16)  # one sum of 15 exact bits and z: one rounding to fp32
    a, b, c = ops.unpack_gemv_q4([w, small, w], [None, None, (1, N)])
    assert torch.equal(a, ref) and torch.equal(c, torch.cat([ref[0::2], ref[1::2]]))
    assert torch.equal(b, Q.weight_values(small).float().to(torch.bfloat16))


# ------------------------------------------------------------------- cache rows

@pytest.mark.parametrize("n_q,n_k,n_v,d", [(12, 1, 2, 128), (15, 5, 5, 64)])
@pytest.mark.parametrize("group,dtype", [(32, torch.bfloat16), (64, torch.float16), (64, torch.bfloat16)])
@pytest.mark.parametrize("n", [1023, 1024, 1501])
def test_append_of_many_tokens(n, n_q, n_k, n_v, d, group, dtype):
    """From 1024 tokens on a wave takes all heads of its token, here in two passes of 8 (d 128) or 16 heads, the last
    not full: codes, scales and queries bit for bit, other rows as they were."""
    g = _gen(n + d)
    B, L = 3, 1600
    qkv = _tokens(g, n, n_q, n_k, n_v, d, dtype)
    pos = torch.randperm(L, generator=g, device="cuda")[:n].int()
    batch = _ints(g, 0, B - 1, n).int()
    table = ops.rope_table(pos, d, 1e6)
    cache = Q.random_cache(g, B, n_k, n_v, L, d, group)
    want = [t.clone() for t in cache]
    q = ops.rope_kv_append_q4(qkv, n_q, table, pos, cache, batch=batch)
    rot, v = _rotate(qkv, table, n_q, n_k, d, torch.float32)
    assert torch.equal(q, rot[:, :n_q].to(dtype))
    for x, kind, at in ((rot[:, n_q:], "k", 0), (v, "v", 2)):
        codes, sz = Q.quantise(x.cpu(), group)
        want[at][batch.long(), :, pos.long()] = Q.pack_row(codes, kind).cuda()
        want[at + 1][batch.long(), :, pos.long()] = sz.cuda()
    assert all(torch.equal(a, b) for a, b in zip(cache, want))
    for name, got in zip(("k", "v"), ops.read_kv_q4(cache, pos, batch, dtype=dtype)):
        held = Q.values(Q.open_row(getattr(cache, name + "_codes")[batch.long(), :, pos.long()], name),
                        getattr(cache, name + "_scales")[batch.long(), :, pos.long()], torch.float32)
        assert torch.equal(got, held.to(dtype))


# ------------------------------------------------------------------- attention

def _score32(x, m):
    """Score and mask as fp32 adds them."""
    return x if m is None else (x.float() + m.float()).double()


def _attention(q, cache, mask, kv_len, scale):
    """Attention in 64 bits and, per output, a bound of the kernel's error before its last rounding, to first order
    in the errors (1 % for the rest).

    A score: at most 32 roundings (18 of a query's sums, 8 of a chain of products, 6 of scales, sums, the factor and
    the mask) of partial sums of q (2 * 16 + c) s and q z; the mask's own rounding where it does not absorb the score,
    which is then exact in both.  An exponential: 2^-22 and 3
    roundings of its argument, at most 8 above the distance from the maximum.  They move the output by what they move
    each weight times the distance of its value from it.  A weight's terms keep 16 bits of p s c; sums over the
    positions take at most 64 roundings (a split is at most two steps of a wave, at most 33 splits) of partial sums of
    p s (2 * 16 + c) and p z."""
    b, q_h, _, d = q.shape
    k, v = Q.cache_values(cache)
    kz, vz = (t.unflatten(-1, (-1, 2)).double() for t in (cache.k_scales, cache.v_scales))
    group, L = d // kz.shape[-2], k.shape[2]
    out, tol = (torch.empty(b, q_h, d, dtype=torch.float64, device=q.device) for _ in range(2))
    for r in range(b):
        n = L if kv_len is None else min(int(kv_len[r]), L)
        for h in range(q_h):
            kh, vh = h * k.shape[1] // q_h, h * v.shape[1] // q_h
            qd, sk, zk = q[r, h, 0].double(), kz[r, kh, :n, :, 0], kz[r, kh, :n, :, 1].abs()
            x = k[r, kh, :n] @ qd * scale
            e = (47 * sk + zk) @ qd.abs().reshape(-1, group).sum(-1) * abs(scale) * 32 * U32
            if mask is not None:
                m = mask[r % mask.shape[0], h % mask.shape[1], 0, :n].double()
                absorbed = m.abs() > 2.0 ** 100  # (scores are below 2^20: half a unit there is 2^75)
                e = torch.where(absorbed | ~m.isfinite(), torch.zeros_like(e), e + 1.001 * m.abs().clamp(max=2.0 ** 20) * U32)
                x = _score32(x, m)
            p = torch.softmax(x, 0)
            o = p @ v[r, vh, :n]
            delta = torch.where(p > 0, e + 2.0 ** -22 + 3 * U32 * ((x - x.max()).abs() + 8), torch.zeros_like(p))
            ps = (p @ vz[r, vh, :n, :, 0]).repeat_interleave(group)
            pz = (p @ vz[r, vh, :n, :, 1].abs()).repeat_interleave(group)
            out[r, h] = o
            tol[r, h] = (1.01 * (p * delta) @ (v[r, vh, :n] - o).abs() + 2.0 ** -17 * 15 * ps
                         + 64 * U32 * (47 * ps + pz + o.abs()))
    return out[:, :, None], tol[:, :, None]


LENS = [4101, 1, 130, 2048, 777, 4100, 3333, 33]
# 8 rows of 4101 positions: 33 splits of 128 for one key head, 26 of 160 for two, so that there are at least 128 blocks
# and a key head's value heads are one unit: two of d 128 (with a mask and groups of 32: units of one), five and two of d 64
UNITS = [(12, 1, 2, 128), (15, 1, 5, 64), (16, 1, 2, 64), (8, 2, 4, 64)]


def _mask(g, b, heads, L, dtype):
    m = _randn(g, b, heads, 1, L)
    m[torch.rand(m.shape, generator=g, device="cuda") < 0.3] = -math.inf
    m[..., 0] = 0
    return m.to(dtype)


@pytest.mark.parametrize("q_h,k_h,v_h,d", UNITS)
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mdt", [None, torch.float32, torch.float16])
def test_units_of_several_value_heads(q_h, k_h, v_h, d, group, dtype, mdt):
    g = _gen(q_h * d + group)
    cache = Q.random_cache(g, len(LENS), k_h, v_h, LENS[0], d, group)
    q = 0.5 * _randn(g, len(LENS), q_h, 1, d)
    q = q.to(dtype)
    kv = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    mask = None if mdt is None else _mask(g, len(LENS), q_h if mdt == torch.float16 else 1, LENS[0], mdt)
    ref, tol = _attention(q, cache, mask, kv, 1 / math.sqrt(d))
    assert float((ref.abs() > 2 * tol).double().mean()) > 0.8  # an output of zeros does not pass
    got = ops.dense_decode_q4(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32)
    _close(got, ref, tol + U32 * ref.abs())
    assert torch.equal(got, ops.dense_decode_q4(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32))


@pytest.mark.parametrize("q_h,k_h,v_h,d", UNITS)
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("masked", [False, True])
def test_units_of_several_value_heads_sum_exactly(q_h, k_h, v_h, d, group, dtype, masked):
    """Queries of zeros weigh every key 1: sums of s c + z, scales 2^-2 .. 2^-4, offsets of at most 1, below 4101 * 143 *
    4 = 2.4 M units of 2^-4, over the number of keys, one rounding."""
    g = _gen(q_h + d + group)
    b, L = len(LENS), LENS[0]
    cache = Q.random_cache(g, b, k_h, v_h, L, d, group)
    cache.v_codes.copy_(_ints(g, 0, 255, *cache.v_codes.shape))
    cache.v_scales[..., 0::2] = (2.0 ** -_ints(g, 2, 4, b, v_h, L, d // group)).half()
    cache.v_scales[..., 1::2] = (_ints(g, -16, 16, b, v_h, L, d // group) / 16).half()
    q = torch.zeros(b, q_h, 1, d, dtype=dtype, device="cuda")
    kv = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    keep = (torch.arange(L, device="cuda") < kv[:, None])[:, None].expand(b, q_h, L)
    mask = None
    if masked:
        hidden = torch.rand(b, q_h, L, generator=g, device="cuda") < 0.4
        hidden[..., 0] = False
        mask = torch.zeros(b, q_h, 1, L, dtype=torch.bfloat16, device="cuda").masked_fill_(hidden[:, :, None], -math.inf)
        keep = keep & ~hidden
    v = Q.cache_values(cache)[1].repeat_interleave(q_h // v_h, 1)
    ref = (torch.matmul(keep.double()[:, :, None], v) / keep.sum(-1)[..., None, None])
    got = ops.dense_decode_q4(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32)
    _close(got, ref, 1.001 * U32 * ref.abs())


@pytest.mark.parametrize("mdt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_h,k_h,v_h,d,group,L", [(15, 1, 5, 64, 32, 517), (12, 1, 2, 128, 64, 517), (15, 1, 5, 64, 64, 4101)])
def test_masks_of_the_lowest_value(mdt, q_h, k_h, v_h, d, group, L):
    """Rows that hide all but five keys, all but the last, and every key with the type's lowest value, which leaves
    the mean of the values where it absorbs the scores; a row of them behind a row's length."""
    g = _gen(L + d)
    b = 8
    cache = Q.random_cache(g, b, k_h, v_h, L, d, group)
    q = (0.5 * _randn(g, b, q_h, 1, d)).to(torch.bfloat16)
    low = torch.finfo(mdt).min
    mask = torch.zeros(b, 1, 1, L, dtype=mdt, device="cuda")
    mask[1, ..., 5:] = low
    mask[2] = low
    mask[3, ..., :-1] = low
    mask[4, ..., : L // 2] = low
    mask[5] = low
    mask[6, ..., 40:] = low
    kv = torch.tensor([L, L, L, L, L, 300, 40, L // 2], dtype=torch.int32, device="cuda")
    ref, tol = _attention(q, cache, mask, kv, 1 / math.sqrt(d))
    assert float((ref.abs() > 2 * tol).double().mean((1, 2, 3)).min()) > 0.6  # in no row do zeros pass
    _close(ops.dense_decode_q4(q, cache, attention_mask=mask, kv_len=kv, out_dtype=torch.float32), ref, tol + U32 * ref.abs())


# ------------------------------------------------------------------- a decoder's cache

def _projected64(m, ids, lo, caches):
    """Per layer the rotated keys and the values [heads, tokens, d] of the tokens ids from position lo on, in 64 bits,
    with attention over the caches; Σ |h| |w| of them in the first layer."""
    s, d, T = m.shape, m.shape.head_dim, len(ids)
    rows, first = [], None
    norm = lambda t: t / (t.square().mean(-1, keepdim=True) + s.eps).sqrt()
    pos = torch.arange(lo, lo + T, device="cuda", dtype=torch.float64)
    ang = pos[:, None] * s.rope_theta ** (-2 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    cs, sn = ang.cos()[:, None], ang.sin()[:, None]
    x = m.embed[ids].double()
    for l in range(s.layers):
        W, h = _weights64(m, m.kw_qkv[l], l, "w_qkv"), norm(x)
        qkv = (h @ W.t() + m.b_qkv[l].double()).view(T, -1, d)
        if l == 0:
            first = (h.abs() @ W.abs().t() + m.b_qkv[l].double().abs()).view(T, -1, d)[:, s.n_q:].transpose(0, 1)
        rot = torch.cat([qkv[..., : d // 2] * cs - qkv[..., d // 2:] * sn, qkv[..., d // 2:] * cs + qkv[..., : d // 2] * sn], -1)
        rows.append((rot[:, s.n_q: s.n_q + s.n_k].transpose(0, 1), qkv[:, s.n_q + s.n_k:].transpose(0, 1)))
        k, v = caches[l]
        o = torch.empty(T, s.n_q, d, dtype=torch.float64, device="cuda")
        at = lo + torch.arange(T, device="cuda")
        for i in range(s.n_q):
            a = rot[:, i] @ k[i * s.n_k // s.n_q].t() / math.sqrt(d)
            a = a.masked_fill(torch.arange(k.shape[1], device="cuda")[None] > at[:, None], -math.inf)
            o[:, i] = torch.softmax(a, -1) @ v[i * s.n_v // s.n_q]
        x = x + o.view(T, -1) @ _weights64(m, m.kw_o[l], l, "w_o").t()
        gate, up = (norm(x) @ _weights64(m, m.kw_gu[l], l, "w_gu").t()).split(s.intermediate, -1)
        x = x + (gate * torch.sigmoid(gate) * up) @ _weights64(m, m.kw_d[l], l, "w_d").t()
    return rows, first


@pytest.mark.parametrize("shape", ["qwen", "llama"])
@pytest.mark.parametrize("weight_bits,batch", [(16, 1), (4, 3), (4, 12)])
def test_decoder_cache_holds_the_tokens_keys_and_values(shape, weight_bits, batch):
    """What a prompt and steps leave in the 4-bit cache against keys and values computed from the weights in 64 bits.
    First layer, element by element: half a step s / 2 beside at most three roundings to bf16 of the projection's
    terms (the normed input, the weight, the result), of both partners where rotated.  Other layers by their norm: a layer rounds to
    bf16 at most 10 times."""
    s = SHAPES[shape]
    m = SagaDecoder(s, batch, 96, mode="dense", kv_bits=4, weight_bits=weight_bits, kv_group=32, keep_source_weights=True,
                    seed=5)
    ids = torch.randint(0, s.vocab, (37,), generator=torch.Generator().manual_seed(8)).cuda()
    m.prefill(ids)
    spans = [(ids, 0)]
    for i in range(3):
        spans.append((m.tokens[-1:].clone(), 37 + i))
        m.step(calibrate=False)
    row = batch - 1
    for tokens, lo in spans:
        hi = lo + len(tokens)
        held = _held(m, row, hi)
        rows, first = _projected64(m, tokens, lo, held)
        for l in range(s.layers):
            cache = m.kv.layer(l)
            for at, (kind, want) in enumerate(zip("kv", rows[l])):
                got = held[l][at][:, lo:hi]
                step = getattr(cache, kind + "_scales")[row, :, lo:hi, 0::2].double().repeat_interleave(32, -1)
                rounding = 0.5 * step.norm() + (10 * l + 3) * 2.0 ** -8 * want.norm()
                assert float((got - want).norm()) <= float(rounding) < 0.6 * float(want.norm()), (l, kind)
                if l == 0:
                    size = first[: s.n_k] if kind == "k" else first[s.n_k:]
                    if kind == "k":
                        size = size + size.roll(s.head_dim // 2, -1)
                    tol = 0.501 * step + 3.05 * 2.0 ** -8 * size
                    assert bool(((got - want).abs() <= tol).all()), kind

