"""A bounded 8-bit decoder whose key heads serve more query heads than one call of attention_weights takes."""
import math
from dataclasses import replace

import pytest
import torch

import test_gpu_kv_decoder as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_q,n_k,n_v", [(20, 1, 2), (40, 2, 4), (17, 1, 1)])
def test_wide_head_groups(monkeypatch, n_q, n_k, n_v):
    """The prompt's weights are those of all its query heads, and steps go on past the cache."""
    monkeypatch.setitem(D.SHAPES, "wide", replace(D.SHAPES["groups"], n_q=n_q, n_k=n_k, n_v=n_v))
    m = D._decoder("wide", 2, 61, True, kv_fp8_block=32, kv_budget=33, kv_recent=8)
    m.prefill(torch.randint(0, m.shape.vocab, (45,), generator=torch.Generator().manual_seed(2)))
    G = math.gcd(n_k, n_v)
    sums = m.kv_weights.sum(-1).double()
    # 32 queries' softmaxes in f32, each off from 1 by at most its 61 + 20 roundings of 2^-24
    assert ((sums - 32 * n_q // G).abs() <= 32 * n_q // G * 81 * 2.0 ** -24 * 2).all()
    for i in range(40):
        token = m.tokens.clone()
        m.step(calibrate=False)
        n = int(m.kv_len[0]) - 1
        ref = D._forward64(m, token[-1:], 45 + i, n - 1, D._held(m, 1, n))
        assert float((m._logits[-1].double() - ref).norm() / ref.norm()) < D._bound(m), i
    assert m._evicted
