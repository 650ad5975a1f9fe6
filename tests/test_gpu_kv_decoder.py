"""SagaDecoder with norms of queries and keys, 8-bit caches and bounded caches on the GPU: a prompt and steps against a
64-bit forward pass that attends over what the caches hold, graphs against eager steps, evictions position by position,
the command line."""
import math
import os
import subprocess
import sys
from dataclasses import replace

import pytest
import torch

import fp8_util as F
import saga_amd.torch_ops  # noqa: F401
from saga_amd import ops
from saga_amd.decoder import DecoderShape, SagaDecoder

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPES = {"qwen": DecoderShape(3, 512, 4, 1, 2, 128, 1024, 2048, 1e6, 1e-6, True),
          "llama": DecoderShape(2, 320, 5, 1, 5, 64, 640, 512, 1e5, 1e-5, False),
          "groups": DecoderShape(2, 512, 8, 2, 4, 64, 640, 512, 1e4, 1e-5, False)}


def _decoder(name, batch, max_len, qk_norm=False, **kw):
    s = replace(SHAPES[name], qk_norm=qk_norm)
    m = SagaDecoder(s, batch, max_len, keep_source_weights=True, seed=5, **{"mode": "dense", **kw})
    g = torch.Generator(device="cuda").manual_seed(11)
    for t in m.q_norm + m.k_norm if qk_norm else ():
        t.copy_(torch.rand(t.shape, generator=g, device="cuda") + 0.5)
    return m


def _norm(x, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def _forward64(m, ids, pos0, place0, caches):
    """Logits of the last of the tokens ids, rotated as positions pos0 .., that see the places up to place0 + their index
    of the caches (per layer k, v [heads, places, d])."""
    s, d, T = m.shape, m.shape.head_dim, len(ids)
    x = m.embed[ids].double()
    pos = torch.arange(pos0, pos0 + T, device="cuda", dtype=torch.float64)
    ang = pos[:, None] * s.rope_theta ** (-2 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    cs, sn = ang.cos()[:, None], ang.sin()[:, None]
    for l in range(s.layers):
        qkv = _norm(x, s.eps) * m.ln1[l].double() @ m.w_qkv[l].double().t() + m.b_qkv[l].double()
        q = qkv.view(T, -1, d)[:, : s.n_q]
        if s.qk_norm:
            q = _norm(q, s.eps) * m.q_norm[l].double()
        q = torch.cat([q[..., : d // 2] * cs - q[..., d // 2:] * sn, q[..., d // 2:] * cs + q[..., : d // 2] * sn], -1)
        k, v = caches[l]
        o = torch.empty(T, s.n_q, d, dtype=torch.float64, device="cuda")
        for h in range(s.n_q):
            a = q[:, h] @ k[h * s.n_k // s.n_q].t() / math.sqrt(d)
            last = place0 + torch.arange(T, device="cuda")
            a = a.masked_fill(torch.arange(k.shape[1], device="cuda")[None] > last[:, None], -math.inf)
            o[:, h] = torch.softmax(a, -1) @ v[h * s.n_v // s.n_q]
        x = x + o.view(T, -1) @ m.w_o[l].double().t()
        gu = _norm(x, s.eps) * m.ln2[l].double() @ m.w_gu[l].double().t()
        g, u = gu.split(s.intermediate, -1)
        x = x + (g * torch.sigmoid(g) * u) @ m.w_d[l].double().t()
    return _norm(x[-1], s.eps) * m.ln_f.double() @ m.lm_head.double().t()


def _values(m):
    """Per layer k, v [batch, heads, places, d] as the caches hold them."""
    if m.kv_fp8_block:
        return [F.cache_values(m.kv.layer(l)) for l in range(m.shape.layers)]
    return [(m.k_cache[l].double(), m.v_cache[l].double()) for l in range(m.shape.layers)]


def _held(m, row, n):
    return [(k[row, :, :n], v[row, :, :n]) for k, v in _values(m)]


def _bound(m):
    """A layer rounds to bf16 at most 10 times (norm, projection, rotation, attention, two residuals, activation, the
    folded weights), each at most half a step, 2^-8, and the head twice more: logits are off by at most this much of
    their size."""
    return (m.shape.layers * 10 + 2) * 2.0 ** -8


@pytest.mark.parametrize("shape", ["qwen", "llama"])
@pytest.mark.parametrize("qk_norm,block", [(True, 0), (False, 64), (True, 32)])
@pytest.mark.parametrize("batch", [1, 3])
def test_decoder_against_64_bits(shape, qk_norm, block, batch):
    m = _decoder(shape, batch, 96, qk_norm, kv_fp8_block=block)
    s, bound = m.shape, _bound(m)
    ids = torch.randint(0, s.vocab, (37,), generator=torch.Generator().manual_seed(1)).cuda()
    m.prefill(ids)
    ref = _forward64(m, ids, 0, 0, _held(m, 0, 37))
    size = float(ref.norm() / math.sqrt(s.vocab))
    assert float(ref[int(m.tokens[0])]) >= float(ref.max()) - 2 * bound * size * 4  # |logits| are within 4 sizes
    for t in m.kv.tensors:  # the prompt in every batch row
        assert all(torch.equal(t[:, 0].contiguous().view(torch.uint8), t[:, i].contiguous().view(torch.uint8))
                   for i in range(batch))
    for i in range(3):
        token = m.tokens.clone()
        m.step(calibrate=False)
        ref = _forward64(m, token[-1:], 37 + i, 37 + i, _held(m, batch - 1, 38 + i))
        assert float((m._logits[-1].double() - ref).norm() / ref.norm()) < bound
    assert m.pos.tolist() == [40] * batch


@pytest.mark.parametrize("mode", ["dense", "atopn", "vanilla"])
@pytest.mark.parametrize("dtype,batch", [(torch.bfloat16, 2), (torch.float16, 2), (torch.bfloat16, 40)])
def test_norms_in_every_mode_graphs_equal_eager(mode, dtype, batch):
    m = _decoder("qwen", batch, 160, True, mode=mode, dtype=dtype, top_n=64)
    ids = torch.randint(0, m.shape.vocab, (90,), generator=torch.Generator().manual_seed(3))
    eager = m.generate(ids, 12, graphs=False)
    assert m._logits.isfinite().all()
    assert all(torch.equal(m.generate(ids, 12), eager) for _ in range(3))


@pytest.mark.parametrize("dtype,batch,weight_bits,block", [(torch.bfloat16, 2, 4, 64), (torch.bfloat16, 40, 16, 128),
                                                           (torch.float16, 2, 16, 32)])
def test_8_bit_graphs_equal_eager(dtype, batch, weight_bits, block):
    m = _decoder("qwen", batch, 128, True, kv_fp8_block=block, dtype=dtype, weight_bits=weight_bits)
    ids = torch.randint(0, m.shape.vocab, (50,), generator=torch.Generator().manual_seed(3))
    eager = m.generate(ids, 12, graphs=False)
    assert m._logits.isfinite().all()
    assert all(torch.equal(m.generate(ids, 12), eager) for _ in range(3))


def test_norms_leave_a_float32_decoder():
    """f32: a norm's result is turned and stored in f32, so steps agree with 64 bits to the f32 products' rounding."""
    m = _decoder("groups", 2, 64, True, dtype=torch.float32)
    ids = torch.randint(0, m.shape.vocab, (20,), generator=torch.Generator().manual_seed(4)).cuda()
    m.prefill(ids)
    token = m.tokens.clone()
    m.step(calibrate=False)
    ref = _forward64(m, token[:1], 20, 20, _held(m, 0, 21))
    # 10 roundings a layer of at most 2^-24, products of up to 640 terms (sums off by at most 640 steps of 2^-24)
    assert float((m._logits[0].double() - ref).norm() / ref.norm()) < 2 * 640 * 2.0 ** -24 * (m.shape.layers * 5 + 1)


@pytest.mark.parametrize("shape,qk_norm", [("qwen", True), ("llama", False), ("groups", True)])
@pytest.mark.parametrize("block,recent", [(0, 8), (32, 0), (64, 33)])
def test_bounded_decoder(shape, qk_norm, block, recent):
    """Steps past the cache: logits against 64 bits over what it holds, each step's weights sum to the heads of a group,
    and an eviction keeps what the gathered weights say."""
    max_len, budget, prompt = 61, 33, 45
    m = _decoder(shape, 2, max_len, qk_norm, kv_fp8_block=block, kv_budget=budget, kv_recent=recent)
    s, bound = m.shape, _bound(m)
    G = math.gcd(s.n_k, s.n_v)
    ids = torch.randint(0, s.vocab, (prompt,), generator=torch.Generator().manual_seed(2)).cuda()
    m.prefill(ids)
    heads = s.n_q // G
    # sums of softmaxes in f32: each is off from 1 by at most its L + 20 roundings of 2^-24
    near = lambda t, want: bool(((t.double() - want).abs() <= want * (max_len + 20) * 2.0 ** -24 * 2).all())
    assert near(m.kv_weights.sum(-1), 32 * heads) and not m.kv_weights[..., prompt:].any()
    n, evictions, gathered = prompt, 0, 32 * heads
    for i in range(75):
        token, full = m.tokens.clone(), n == max_len
        weights, held = m.kv_weights.clone(), _values(m)
        m.step(calibrate=False)
        if full:
            evictions += 1
            for l in range(s.layers):
                for b in range(2):
                    for u in range(G):
                        kept = F.kept_positions(weights[l, b, u].tolist(), n, budget, recent)
                        for t, now in zip(held[l], _values(m)[l]):
                            hs = t.shape[1] // G
                            rows = now[b, u * hs:(u + 1) * hs, :budget]
                            want = t[b, u * hs:(u + 1) * hs, kept]
                            if not block:
                                assert torch.equal(rows, want)
                            else:  # a larger scale of the place's block: off by at most its half step, 2^-10 s
                                c = m.kv.layer(l)
                                sc = (c.k_scales if t is held[l][0] else c.v_scales)[b, u * hs:(u + 1) * hs].double()
                                half = sc.repeat_interleave(block, 1)[:, :budget, None] * 2.0 ** -10
                                # the step's own token may have set the last block's scale anew: 2^-4 of a value
                                assert bool(((rows - want).abs() <= 2 * half + want.abs() * 2.0 ** -4).all())
            n = budget
        n += 1
        ref = _forward64(m, token[-1:], prompt + i, n - 1, _held(m, 1, n))
        assert float((m._logits[-1].double() - ref).norm() / ref.norm()) < bound, i
        assert not m.kv_weights[..., n:].any()
        if not evictions:
            gathered += heads
            assert near(m.kv_weights.sum(-1), gathered)
    assert evictions == 3 and m.pos.tolist() == [prompt + 75] * 2 and m.slot.tolist() == [n] * 2
    with pytest.raises(RuntimeError, match="evicted"):
        m.reset()
    m.prefill(ids)
    assert m.pos.tolist() == [prompt] * 2 and m.slot.tolist() == [prompt] * 2


@pytest.mark.parametrize("block,dtype,weight_bits", [(0, torch.bfloat16, 16), (32, torch.float16, 16), (64, torch.bfloat16, 4),
                                                     (0, torch.float32, 16)])
def test_bounded_graphs_equal_eager(block, dtype, weight_bits):
    m = _decoder("qwen", 2, 80, True, kv_fp8_block=block, kv_budget=50, kv_recent=10, dtype=dtype, weight_bits=weight_bits)
    ids = torch.randint(0, m.shape.vocab, (60,), generator=torch.Generator().manual_seed(6))
    eager = m.generate(ids, 130, graphs=False)
    assert m._logits.isfinite().all()
    assert all(torch.equal(m.generate(ids, 130), eager) for _ in range(2))


def test_a_cache_that_never_fills_is_an_unbounded_one():
    """The same tokens with and without a budget until the cache is full."""
    ids = torch.randint(0, 2048, (40,), generator=torch.Generator().manual_seed(7))
    for block in (0, 64):
        a = _decoder("qwen", 2, 80, True, kv_fp8_block=block)
        b = _decoder("qwen", 2, 80, True, kv_fp8_block=block, kv_budget=50, kv_recent=10)
        assert torch.equal(a.generate(ids, 40), b.generate(ids, 40))
        assert all(torch.equal(x, y) for x, y in zip(a.kv.tensors, b.kv.tensors))


@pytest.mark.parametrize("block", [32, 128])
def test_fill_synthetic_8_bits(block):
    m = _decoder("llama", 2, 5000, kv_fp8_block=block, kv_budget=4900)
    m.fill_synthetic(4500)
    # 2 x 4500 x 64 normal values per head: mean within 6 / sqrt(n), deviation within 2 % (rounding adds 0.1 % of variance)
    for t in F.cache_values(m.kv.layer(1)):
        x = t[:, :, :4500]
        assert abs(float(x.mean())) < 6 / math.sqrt(x.numel()) and abs(float(x.std()) - 1) < 0.02
        assert not t[:, :, 4500:].any()
    m.capture()
    m.replay(0)
    torch.cuda.synchronize()
    assert m._logits.isfinite().all() and int(m.pos[0]) == 4501 and int(m.slot[0]) == 4501


def test_traced_programs_equal_eager_ones():
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = F.random_cache(g, 2, 1, 2, 700, 128, 64)
    q = torch.randn(2, 12, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    mask = torch.zeros(2, 1, 1, 700, device="cuda").masked_fill_(torch.arange(700, device="cuda") < 9, -math.inf)
    kv = torch.tensor([700, 333], dtype=torch.int32, device="cuda")
    torch.library.opcheck(torch.ops.saga.dense_decode_fp8, (q, *cache, mask, 0.1, kv))

    def program(x):
        return 2 * torch.ops.saga.dense_decode_fp8(x + 1, *cache, mask, None, kv)

    got = torch.compile(program, backend="aot_eager", fullgraph=True)(q)
    assert torch.equal(got, 2 * ops.dense_decode_fp8(q + 1, cache, attention_mask=mask, kv_len=kv))


def test_command_line(tmp_path):
    pytest.importorskip("transformers")
    from ckpt_util import save_saga_checkpoint, tiny_hf_model
    path = str(tmp_path / "saga")
    save_saga_checkpoint(tiny_hf_model("qwen2", n_kv=2, n_k_shared=1, tie=True, d=64, intermediate=512, vocab=1024),
                         path, n_k=1)
    cmd = [sys.executable, "-m", "saga_amd.speedup", "--model_path", path, "--attention", "full", "--batch_sizes", "2",
           "--seq_lengths", "200", "--num_new_tokens", "4", "--num_warmup", "1", "--num_iterations", "2", "--timeout",
           "100", "--cuda_graph", "--kv_fp8_block", "64"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=110, cwd=ROOT)
    print(r.stdout[-2000:], r.stderr[-2000:], flush=True)
    assert r.returncode == 0 and "SUMMARY" in r.stdout and "FAILED" not in r.stdout
