"""SagaDecoder over 8-bit caches on the GPU: reset() rewinds to just after the prompt, whatever the steps behind it did to
the scale of the block that the prompt ends inside."""
import pytest
import torch

from test_gpu_kv_decoder import _decoder

pytestmark = pytest.mark.gpu


def _steps(m, n, graphs):
    """Tokens and logits of n steps, and what the caches hold behind them: rows, and scales of blocks that are begun."""
    out = []
    for i in range(n):
        if graphs:
            m.replay(i)
        else:
            m.step(calibrate=False)
        out += [m.tokens.clone(), m._logits.clone()]
    end = int(m.kv_len[0]) - 1
    blocks = -(-end // m.kv_fp8_block)
    return out + [t[..., :end, :].clone() if t.dtype == torch.uint8 else t[..., :blocks].clone() for t in m.kv.tensors]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("block,prompt", [(32, 37), (64, 127), (128, 40), (32, 64)])
@pytest.mark.parametrize("batch,qk_norm,budget,graphs", [(1, False, 0, False), (3, True, 0, False), (2, False, 100, False),
                                                         (2, False, 0, True), (2, True, 100, True)])
@pytest.mark.parametrize("synthetic", [False, True])
def test_reset_undoes_a_raised_scale(block, prompt, batch, qk_norm, budget, graphs, synthetic):
    m = _decoder("qwen", batch, 160, qk_norm, kv_fp8_block=block, kv_budget=budget)
    if synthetic:
        m.fill_synthetic(prompt)
    else:
        m.prefill(torch.randint(0, m.shape.vocab, (prompt,), generator=torch.Generator().manual_seed(1)))
    held = [t.clone() for t in m.kv.tensors]
    if graphs:
        m.capture()
    first = _steps(m, 5, graphs)
    m.reset()
    biases = [b.clone() for b in m.b_qkv]
    for b in m.b_qkv:  # keys (without norms) and values of thousands beside the prompt's
        b.mul_(2.0 ** 18)
    _steps(m, 2, graphs)
    at = prompt // block
    for t, h in zip(m.kv.tensors[1::2] if not qk_norm else m.kv.tensors[3:], held[1::2] if not qk_norm else held[3:]):
        assert bool((t[..., at] > h[..., at]).all())  # the scale of the block was raised
    for b, was in zip(m.b_qkv, biases):
        b.copy_(was)
    m.reset()
    for t, h in zip(m.kv.tensors, held):
        end = prompt if t.dtype == torch.uint8 else -(-prompt // block)
        view = (lambda x: x[..., :end, :]) if t.dtype == torch.uint8 else (lambda x: x[..., :end])
        assert torch.equal(view(t), view(h))
    assert _same(_steps(m, 5, graphs), first)
    m.reset()
    assert _same(_steps(m, 5, graphs), first)


def test_a_prompt_after_another():
    """What a shorter or longer prompt leaves to rewind to is its own."""
    m, ref = (_decoder("qwen", 2, 160, False, kv_fp8_block=64) for _ in range(2))
    ids = torch.randint(0, m.shape.vocab, (100,), generator=torch.Generator().manual_seed(2))
    m.prefill(ids)
    _steps(m, 3, False)
    m.prefill(ids[:70])
    ref.prefill(ids[:70])
    want = _steps(ref, 4, False)
    assert _same(_steps(m, 4, False), want)
    m.reset()
    assert _same(_steps(m, 4, False), want)
