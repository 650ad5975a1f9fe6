"""Limits of the 8-bit forms on the GPU: what the attention holds of a weight, norms of keys beside large and small
magnitudes."""
import pytest
import torch

import fp8_util as F
from saga_amd import ops
from test_gpu_fp8 import _append_reference, _keys

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_h,k_h,v_h,d", [(12, 1, 2, 128), (12, 2, 2, 128), (15, 1, 5, 64), (15, 5, 5, 64), (16, 1, 8, 64)])
def test_a_weight_keeps_24_bits(q_h, k_h, v_h, d, dtype):
    """Two positions, the first of score 0 and value 0, the second of an exact score x from -2 to -1/4: outputs are
    v e^x / (1 + e^x).  The exponential's argument x log2(e) is rounded and log2(e) itself (3 and 1.5 of 2^-24 of the
    result, |x| <= 2), the instruction is off by a step (2 of them), the sum of the weights, the products' sums of three
    terms, the join and the division by one each, 12 in all: within 24 half steps."""
    b = 130  # (so many rows that several value heads make a unit)
    g = _gen(q_h + d)
    q = torch.zeros(b, q_h, 1, d, device="cuda")
    q[..., 0] = 0.5 + 0.5 * torch.rand(b, q_h, 1, generator=g, device="cuda")
    q = q.to(dtype)
    k, v = torch.zeros(b, k_h, 2, d, device="cuda"), torch.zeros(b, v_h, 2, d, device="cuda")
    k[:, :, 1, 0] = -(0.5 + 1.5 * torch.rand(b, k_h, generator=g, device="cuda"))
    v[:, :, 1] = torch.randn(b, v_h, d, generator=g, device="cuda")
    k, v = (t.to(torch.float8_e4m3fn) for t in (k, v))
    ones = [torch.ones(b, h, 1, device="cuda") for h in (k_h, v_h)]
    cache = ops.KVFP8(k.view(torch.uint8), ones[0], v.view(torch.uint8), ones[1], 32)
    x = q[:, :, 0, 0].double() * k[:, :, 1, 0].double().repeat_interleave(q_h // k_h, 1)
    assert float(x.max()) <= -0.25 and float(x.min()) >= -2.0
    p = torch.exp(x) / (1 + torch.exp(x))
    ref = p[..., None] * v[:, :, 1].double().repeat_interleave(q_h // v_h, 1)
    got = ops.dense_decode_fp8(q, cache, scaling=1.0, out_dtype=torch.float32)[:, :, 0].double()
    assert ((got - ref).abs() <= 24 * U32 * ref.abs()).all(), float(((got - ref).abs() / ref.abs().clamp(min=1e-30)).max() / U32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 128)])
@pytest.mark.parametrize("each", [1, 45])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("aligned", [True, False])
def test_normed_keys_of_any_magnitude(dtype, d, block, each, eps, aligned):
    """Keys of magnitudes 2^-80 to 2^120, whose squares leave a float's range, in 16-byte rows and in others: codes and
    scales of the formula in 64 bits, bit by bit."""
    n_q, n_k, n_v, b = 2, 5, 1, 3
    g = _gen(d + each)
    cache = F.random_cache(g, b, n_k, n_v, 200, d, block)
    n = b * each
    size = torch.tensor([1.0] * n_q + [2.0 ** e for e in (70, 120, -80, 63.5, 0)] + [1.0], device="cuda")
    x = torch.randn(n, n_q + n_k + n_v, d, generator=g, device="cuda") * size[:, None]
    if each == 1:  # one large value in a head of small ones
        x[:, n_q + n_k - 1, 5] = 2.0 ** 66
    wide = torch.zeros(n, (n_q + n_k + n_v) * d + 8, dtype=dtype, device="cuda")
    qkv = wide[:, :-8] if aligned else wide[:, 1:-7]
    qkv.copy_(x.flatten(1))
    assert qkv.isfinite().all()
    start = [7, block, 40]
    pos = torch.cat([torch.arange(each) + p for p in start]).int().cuda()
    table = ops.rope_table(pos, d, 1e4)
    norms = [(0.5 + torch.rand(d, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    k, v = _keys(qkv, table, n_q, n_k, d, norms[1], eps), qkv.double().reshape(n, -1, d)[:, n_q + n_k:]
    want = _append_reference(cache, k, v, start, [each] * b)
    ops.norm_rope_kv_append_fp8(qkv, n_q, table, torch.tensor(start, device="cuda").int(), cache, *norms, eps=eps)
    assert F.same(cache, want)
    held = F.cache_values(cache)[0][0, :, 7]
    # (with eps the head of 2^-80 is 2^-70 beside a held block's normal values: zeros, as in the reference)
    assert held.isfinite().all() and (held.abs().amax(-1) > 0)[[0, 1, 3, 4] if eps else slice(None)].all()
