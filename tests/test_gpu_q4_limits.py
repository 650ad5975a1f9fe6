"""Limits of the 4-bit forms on the GPU: values at the end of the range of f16, long sums, the memory of a decoder's
construction."""
import pytest
import torch

import q4_util as Q
from saga_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_values_at_the_end_of_the_f16_range_stay_finite(d, group):
    """A scale is rounded up, so that a group from -60000 to 65504 (z -60000, s 8368, c 15) reads as 65520, which f16
    would round to infinity: reads and attention of f16 stay at 65504."""
    g = torch.Generator(device="cuda").manual_seed(d + group)
    n, L = 3, 700
    x = (torch.rand(n, 3, d, generator=g, device="cuda") * 100000 - 50000).half().float()
    x[..., ::8], x[..., 3::8] = -60000.0, 65504.0
    held = Q.values(*_grouped(x, group), torch.float32)
    assert float(held.max()) == 65520.0 and not held.half().isfinite().all()
    cache = Q.random_cache(g, n, 1, 1, L, d, group)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    table = torch.tensor([1.0, 0.0], device="cuda").expand(n, d // 2, 2).contiguous()  # no rotation
    ops.rope_kv_append_q4(x.flatten(1).half(), 1, table, pos, cache)
    for got, want in zip(ops.read_kv_q4(cache, pos, dtype=torch.float16), (held[:, 1:2], held[:, 2:3])):
        assert torch.equal(got, want.clamp(max=65504.0).half())
    for got, want in zip(ops.read_kv_q4(cache, pos, dtype=torch.float32), (held[:, 1:2], held[:, 2:3])):
        assert torch.equal(got, want)
    # attention over the one key that the mask leaves, in one block and in several splits; over none of them NaN
    for length in (3, L):
        part = ops.KVQ4(*(t[:, :, :length].contiguous() for t in cache))
        mask = torch.full((n, 1, 1, length), float("-inf"), device="cuda")
        for i in range(n - 1):
            mask[i, 0, 0, i] = 0
        for dtype in (torch.float16, torch.bfloat16):
            q = torch.zeros(n, 2, 1, d, dtype=dtype, device="cuda")
            out = ops.dense_decode_q4(q, part, attention_mask=mask, out_dtype=torch.float16)[:, :, 0]
            want = held[:, 2].clamp(max=65504.0)
            # a weight's terms keep 16 bits of p s c, the offset and the sums 2^-20 of p s (128 + c)
            tol = 2.0 ** -11 * want.abs() + 2.0 ** -17 * 15 * 8368 + 2.0 ** -20 * 143 * 8368
            assert bool(((out[:-1].float() - want[:-1, None]).abs() <= tol[:-1, None]).all())
            assert out[:-1].isfinite().all() and out[-1].isnan().all()
    cache.v_scales[0, 0, 0, 0] = float("inf")  # what is infinite stays so
    assert not ops.read_kv_q4(cache, pos, dtype=torch.float16)[1][0, 0, :group].isfinite().any()


def _grouped(x, group):
    codes, sz = Q.quantise(x.cpu(), group)
    return codes.cuda(), sz.cuda()


@pytest.mark.parametrize("group", [32, 64])
def test_long_sums_are_equally_exact_in_every_dim(group):
    """Over 33000 positions what is added to the codes on their way to the products grows and cancels: the rounding of
    these sums has to be the same in all dims.  Root mean square errors of the tiles of 16 dims, over 96 heads of other
    queries: a head's dims share terms, so each is known to some 1 / sqrt(2 * 96), 7 %, and they lie within a factor of 2."""
    g = torch.Generator(device="cuda").manual_seed(group)
    b, q_h, L, d = 8, 12, 33000, 128
    cache = Q.random_cache(g, b, 1, 2, L, d, group)
    q = torch.randn(b, q_h, 1, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = Q.cache_values(cache)
    p = torch.softmax(torch.matmul(q.double()[:, :, 0], k[:, 0].transpose(1, 2).contiguous()) / 16, -1)
    ref = torch.matmul(p.view(b, 2, q_h // 2, L), v).reshape(b, q_h, d)
    got = ops.dense_decode_q4(q, cache, scaling=1 / 16, out_dtype=torch.float32)[:, :, 0].double()
    rms = (got - ref).square().mean((0, 1)).view(d // 16, 16).mean(1).sqrt()
    print([f"{float(r):.1e}" for r in rms], flush=True)
    assert float(rms.max()) < 2 * float(rms.min())


def test_a_decoder_is_built_within_its_planned_memory():
    """Construction needs the source weights, the 4-bit copies, caches and workspaces that the planner counts, and
    one weight's temporaries at a time: not the norm-folded bf16 copies of all layers (35 MB a layer here)."""
    from saga_amd.decoder import DecoderShape, SagaDecoder
    from saga_amd.kv_cache import plan_capacity
    s = DecoderShape(40, 1024, 8, 1, 2, 64, 8192, 2048, 1e6, 1e-6, True)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    m = SagaDecoder(s, 4, 512, mode="dense", kv_bits=4, weight_bits=4)
    peak = torch.cuda.max_memory_allocated() - before
    plan = plan_capacity(s, batch=4, budget_bytes=1 << 37, kv_bits=4, weight_bits=4)
    planned = plan.weight_bytes + plan.workspace_bytes + m.kv.nbytes
    one = 4 * 2 * s.intermediate * s.hidden  # the largest weight in fp32
    print(f"peak {peak / 1e6:.0f} MB, planned {planned / 1e6:.0f} MB, one weight {one / 1e6:.0f} MB", flush=True)
    assert peak <= planned + 8 * one < planned + 40 * 35e6
