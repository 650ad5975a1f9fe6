"""dense_decode_q4 as a torch.library operator: its fake implementation (CPU), and on the GPU its checks and a program
compiled around it."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import q4_util as Q
import saga_amd.torch_ops  # noqa: F401
from saga_amd import ops


def test_fake_implementation_gives_the_output_shape():
    with FakeTensorMode():
        for b, q_h, k_h, v_h, L, d, group in ((2, 12, 1, 2, 300, 128, 64), (1, 15, 5, 5, 40, 64, 32)):
            q = torch.empty(b, q_h, 1, d, dtype=torch.float16, device="cuda")
            parts = [torch.empty(b, h, L, n, dtype=dt, device="cuda") for h in (k_h, v_h)
                     for n, dt in ((d // 2, torch.uint8), (2 * d // group, torch.float16))]
            out = torch.ops.saga.dense_decode_q4(q, *parts)
            assert out.shape == (b, q_h, 1, d) and out.dtype == torch.float16 and out.device.type == "cuda"
    schema = torch.ops.saga.dense_decode_q4.default._schema
    assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments)


@pytest.mark.gpu
def test_traced_programs_equal_eager_ones():
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = Q.random_cache(g, 2, 1, 2, 700, 128, 64)
    q = torch.randn(2, 12, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    mask = torch.zeros(2, 1, 1, 700, device="cuda").masked_fill_(torch.arange(700, device="cuda") < 9, -math.inf)
    kv = torch.tensor([700, 333], dtype=torch.int32, device="cuda")
    torch.library.opcheck(torch.ops.saga.dense_decode_q4, (q, *cache, mask, 0.1, kv))

    def program(x):
        return 2 * torch.ops.saga.dense_decode_q4(x + 1, *cache, mask, None, kv)

    got = torch.compile(program, backend="aot_eager", fullgraph=True)(q)
    assert torch.equal(got, 2 * ops.dense_decode_q4(q + 1, cache, attention_mask=mask, kv_len=kv))
