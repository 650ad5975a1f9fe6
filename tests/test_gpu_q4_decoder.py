"""SagaDecoder with 4-bit caches and 4-bit weights on the GPU: a prompt and steps against a 64-bit forward pass that
attends over what the caches hold, graphs against eager steps, the command line."""
import math
import os
import subprocess
import sys

import pytest
import torch

import q4_util as Q
from saga_amd.decoder import DecoderShape, SagaDecoder

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPES = {"qwen": DecoderShape(3, 512, 4, 1, 2, 128, 1024, 2048, 1e6, 1e-6, True),
          "llama": DecoderShape(2, 320, 5, 1, 5, 64, 640, 512, 1e5, 1e-5, False)}


def _weights64(m, w, layer, name):
    """A projection as the step computes it: 64-bit values of its 4-bit form, or the source weight with its norm."""
    if m.weight_bits == 4:
        W = Q.weight_values(w)
        if name == "w_gu":
            W = torch.cat([W[0::2], W[1::2]])
        return W
    W = getattr(m, name)[layer].double() if layer is not None else m.lm_head.double()
    norm = {"w_qkv": m.ln1, "w_gu": m.ln2}.get(name)
    return W * norm[layer].double() if norm is not None else W * m.ln_f.double() if layer is None else W


def _forward64(m, ids, lo, caches):
    """Logits of the last of the tokens ids (positions 0 ..), keys and values of positions >= lo and below as the
    caches (per layer k, v [heads, positions, d]) hold them."""
    s, d, T = m.shape, m.shape.head_dim, len(ids)
    x = m.embed[ids].double()
    pos = torch.arange(lo, lo + T, device="cuda", dtype=torch.float64)
    ang = pos[:, None] * s.rope_theta ** (-2 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    cs, sn = ang.cos()[:, None], ang.sin()[:, None]
    norm = lambda t: t / (t.square().mean(-1, keepdim=True) + s.eps).sqrt()
    for l in range(s.layers):
        qkv = norm(x) @ _weights64(m, m.kw_qkv[l], l, "w_qkv").t() + m.b_qkv[l].double()
        q = qkv.view(T, -1, d)[:, : s.n_q]
        q = torch.cat([q[..., : d // 2] * cs - q[..., d // 2:] * sn, q[..., d // 2:] * cs + q[..., : d // 2] * sn], -1)
        k, v = caches[l]
        o = torch.empty(T, s.n_q, d, dtype=torch.float64, device="cuda")
        for h in range(s.n_q):
            a = q[:, h] @ k[h * s.n_k // s.n_q].t() / math.sqrt(d)
            a = a.masked_fill(torch.arange(k.shape[1], device="cuda")[None] > (lo + torch.arange(T, device="cuda"))[:, None],
                              -math.inf)
            o[:, h] = torch.softmax(a, -1) @ v[h * s.n_v // s.n_q]
        x = x + o.view(T, -1) @ _weights64(m, m.kw_o[l], l, "w_o").t()
        gu = norm(x) @ _weights64(m, m.kw_gu[l], l, "w_gu").t()
        g, u = gu.split(s.intermediate, -1)
        x = x + (g * torch.sigmoid(g) * u) @ _weights64(m, m.kw_d[l], l, "w_d").t()
    return norm(x[-1]) @ _weights64(m, m.kw_lm, None, "lm").t()


def _held(m, row, n):
    if m.kv_bits == 4:
        out = [Q.cache_values(m.kv.layer(l)) for l in range(m.shape.layers)]
    else:
        out = [(m.k_cache[l].double(), m.v_cache[l].double()) for l in range(m.shape.layers)]
    return [(k[row, :, :n], v[row, :, :n]) for k, v in out]


@pytest.mark.parametrize("shape", ["qwen", "llama"])
@pytest.mark.parametrize("kv_bits,weight_bits", [(4, 16), (16, 4), (4, 4)])
@pytest.mark.parametrize("batch", [1, 3])
def test_decoder_against_64_bits(shape, kv_bits, weight_bits, batch):
    """A layer rounds to bf16 at most 10 times (norm, projection, rotation, attention, two residuals, activation, the
    opened weights), each at most half a step, 2^-8: logits are off by at most layers * 10 * 2^-8 of their size."""
    s = SHAPES[shape]
    m = SagaDecoder(s, batch, 96, mode="dense", kv_bits=kv_bits, weight_bits=weight_bits, kv_group=32,
                    keep_source_weights=True, seed=5)
    bound = (s.layers * 10 + 2) * 2.0 ** -8
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, s.vocab, (37,), generator=g).cuda()
    m.prefill(ids)
    ref = _forward64(m, ids, 0, _held(m, 0, 37))
    size = float(ref.norm() / math.sqrt(s.vocab))
    first = int(m.tokens[0])
    assert float(ref[first]) >= float(ref.max()) - 2 * bound * size * 4  # |logits| are within 4 sizes
    for t in m.kv.tensors:  # the prompt in every batch row, nothing behind it
        assert all(torch.equal(t[:, 0].view(torch.uint8), t[:, i].view(torch.uint8)) for i in range(batch))
        assert not t[:, :, :, 37:].any()
    for i in range(3):
        token = m.tokens.clone()
        m.step(calibrate=False)
        ref = _forward64(m, token[-1:], 37 + i, _held(m, batch - 1, 38 + i))
        assert float((m._logits[-1].double() - ref).norm() / ref.norm()) < bound
    assert m.pos.tolist() == [40] * batch


@pytest.mark.parametrize("dtype,batch,weight_bits", [(torch.bfloat16, 2, 4), (torch.bfloat16, 40, 16), (torch.float16, 2, 16)])
def test_decoder_graphs_equal_eager(dtype, batch, weight_bits):
    s = SHAPES["qwen"]
    m = SagaDecoder(s, batch, 128, mode="dense", kv_bits=4, weight_bits=weight_bits, dtype=dtype, seed=2)
    ids = torch.randint(0, s.vocab, (50,), generator=torch.Generator().manual_seed(3))
    eager = m.generate(ids, 12, graphs=False)
    assert torch.equal(m.generate(ids, 12), eager) and torch.equal(m.generate(ids, 12), eager)


@pytest.mark.parametrize("batch", [1, 8, 32])
def test_atopn_with_4_bit_weights(batch):
    """4-bit weights beside Atop-N attention over 16-bit caches."""
    s = SHAPES["qwen"]
    m = SagaDecoder(s, batch, 2048, mode="atopn", top_n=256, weight_bits=4, seed=4)
    ids = torch.randint(0, s.vocab, (1500,), generator=torch.Generator().manual_seed(6))
    eager = m.generate(ids, 10, graphs=False)
    assert m._logits.isfinite().all()
    assert all(torch.equal(m.generate(ids, 10), eager) for _ in range(3))


def test_fill_synthetic_q4():
    s = SHAPES["llama"]
    m = SagaDecoder(s, 2, 5000, mode="dense", kv_bits=4, weight_bits=4)
    m.fill_synthetic(4500)
    k, v = Q.cache_values(m.kv.layer(1))
    # 2 x 4500 x 64 normal values per head: mean within 6 / sqrt(n), deviation within 2 % (quantisation adds 0.8 % of variance)
    for t in (k, v):
        x = t[:, :, :4500]
        assert abs(float(x.mean())) < 6 / math.sqrt(x.numel()) and abs(float(x.std()) - 1) < 0.02
        assert not t[:, :, 4500:].any()
    m.capture()
    m.replay(0)
    torch.cuda.synchronize()
    assert m._logits.isfinite().all() and int(m.pos[0]) == 4501


def test_command_line(tmp_path):
    pytest.importorskip("transformers")
    from ckpt_util import save_saga_checkpoint, tiny_hf_model
    path = str(tmp_path / "saga")
    save_saga_checkpoint(tiny_hf_model("qwen2", n_kv=2, n_k_shared=1, tie=True, d=64, intermediate=512, vocab=1024),
                         path, n_k=1)
    cmd = [sys.executable, "-m", "saga_amd.speedup", "--model_path", path, "--attention", "full", "--batch_sizes", "2",
           "--seq_lengths", "200", "--num_new_tokens", "4", "--num_warmup", "1", "--num_iterations", "2", "--timeout",
           "100", "--cuda_graph", "--kv_bits", "4", "--weight_bits", "4"]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=110, cwd=ROOT)
    print(r.stdout[-2000:], r.stderr[-2000:], flush=True)
    assert r.returncode == 0 and "SUMMARY" in r.stdout and "FAILED" not in r.stdout
