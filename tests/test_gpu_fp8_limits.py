"""Limits of the 8-bit forms on the GPU: what the attention holds of a weight."""
import pytest
import torch

from saga_amd import ops

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
