"""Bounded decoders on the CPU: head groups that are refused when the decoder is built, not at its first step, and what
the planner counts for one."""
import math
from dataclasses import replace

import pytest
import torch

from saga_amd import _lib
from saga_amd.decoder import QWEN25_15B_SAGA, DecoderShape, SagaDecoder
from saga_amd.kv_cache import decode_weight_bytes, decode_workspace_bytes, kv_cache_bytes, plan_capacity

TINY = DecoderShape(2, 64, 4, 1, 2, 64, 128, 256, 1e4, 1e-6)


@pytest.mark.parametrize("n_q,n_k", [(18, 1), (34, 2), (40, 2)])
def test_wide_head_groups_of_16_bit_caches_are_refused(n_q, n_k):
    wide = replace(TINY, n_q=n_q, n_k=n_k)
    with pytest.raises(ValueError, match="16 query heads per key head"):
        SagaDecoder(wide, 1, 16, mode="dense", device="cpu", kv_budget=8)
    SagaDecoder(wide, 1, 16, mode="dense", device="cpu", kv_budget=8, kv_fp8_block=32)
    SagaDecoder(replace(wide, n_q=16 * n_k), 1, 16, mode="dense", device="cpu", kv_budget=8)


@pytest.mark.parametrize("block,dtype", [(0, torch.bfloat16), (0, torch.float32), (64, torch.bfloat16)])
def test_plans_count_what_a_bounded_decoder_holds(block, dtype):
    lib, b, L, keep, recent = _lib.load(), 3, 300, 200, 20
    s = replace(TINY, n_q=8, n_k=2, n_v=4, layers=3)
    m = SagaDecoder(s, b, L, mode="dense", device="cpu", dtype=dtype, kv_fp8_block=block, kv_budget=keep, kv_recent=recent)
    G, row = math.gcd(s.n_k, s.n_v), s.head_dim if block else s.head_dim * m.k_cache.element_size()
    held = sum(t.numel() * t.element_size() for t in (m.kv_weights, m._prompt_weights))
    assert held == 2 * 4 * s.layers * b * G * L
    more = lib.saga_evict_workspace_bytes(b, G, keep, recent, s.n_k + s.n_v, row, 1) + held
    if block:
        more += lib.saga_dense_fp8_workspace_bytes(b, s.n_q, L, 64, 1) - lib.saga_dense_fp8_workspace_bytes(b, s.n_q, L, 64, 0)
    else:
        more += lib.saga_attention_weights_workspace_bytes(b, s.n_q, s.n_k, L)
    args = dict(kv_fp8_block=block, dtype=dtype)
    assert decode_workspace_bytes(s, b, L, 512, **args, kv_budget=keep, kv_recent=recent) == \
        decode_workspace_bytes(s, b, L, 512, **args) + more
    norms = decode_weight_bytes(replace(s, qk_norm=True), dtype) - decode_weight_bytes(s, dtype)
    assert norms == 2 * s.layers * s.head_dim * m.embed.element_size()


def test_plans_of_bounded_caches():
    s, budget = QWEN25_15B_SAGA, 20 * 10**9
    for block in (0, 64):
        free, bound = (plan_capacity(s, batch=8, budget_bytes=budget, kv_fp8_block=block, **kw)
                       for kw in ({}, dict(kv_budget=4096, kv_recent=64)))
        assert bound.max_len < free.max_len and bound.total_bytes <= budget * 0.95
        assert bound.kv_bytes == kv_cache_bytes(s, 8, bound.max_len, fp8_block=block)
        assert bound.workspace_bytes == decode_workspace_bytes(s, 8, bound.max_len, 512, kv_fp8_block=block, kv_budget=4096,
                                                               kv_recent=64)
        with pytest.raises(MemoryError, match="kv_budget"):
            plan_capacity(s, batch=8, budget_bytes=budget, kv_fp8_block=block, kv_budget=free.max_len)
        assert plan_capacity(s, max_len=8192, budget_bytes=budget, kv_fp8_block=block, kv_budget=4096).batch >= 8
    for kw, needle in ((dict(kv_budget=512, kv_bits=4), "16- or 8-bit caches"), (dict(kv_budget=8192), "max_len - 1"),
                       (dict(kv_budget=64, kv_recent=65), "kv_recent"), (dict(kv_recent=4), "kv_budget")):
        with pytest.raises(ValueError, match=needle):
            plan_capacity(s, max_len=8192, budget_bytes=budget, **kw)
    with pytest.raises(ValueError, match="16 query heads"):
        plan_capacity(replace(s, n_q=20), max_len=8192, budget_bytes=budget, kv_budget=64)
