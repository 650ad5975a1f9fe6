"""What the planner, the decoder, the checkpoint loader and the command line say about 8-bit caches, norms of queries and
keys and bounded caches (CPU)."""
import subprocess
from dataclasses import replace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import saga_amd.torch_ops  # noqa: F401
from saga_amd import _lib, speedup
from saga_amd.decoder import QWEN25_15B_SAGA, DecoderShape, SagaDecoder
from saga_amd.kv_cache import HBM_BYTES_MI355X, KVCache, decode_workspace_bytes, kv_cache_bytes, plan_capacity

TINY = DecoderShape(2, 64, 4, 1, 2, 64, 128, 256, 1e4, 1e-6)


def test_plans_are_decoders_that_can_be_built():
    for shape, kw, needle in (
            (TINY, dict(kv_fp8_block=16), "blocks of 32, 64 or 128"), (TINY, dict(kv_fp8_block=8), "blocks of 32"),
            (replace(TINY, head_dim=32), dict(kv_fp8_block=64), "head dim"),
            (TINY, dict(kv_fp8_block=64, dtype=torch.float32), "bf16 or f16"),
            (TINY, dict(kv_fp8_block=64, kv_bits=4), "exclude each other"),
            (replace(TINY, qk_norm=True), dict(kv_bits=4), "norms of queries and keys"),
            (replace(TINY, qk_norm=True, head_dim=32), {}, "norms of queries and keys")):
        with pytest.raises(ValueError, match=needle):
            plan_capacity(shape, batch=2, budget_bytes=HBM_BYTES_MI355X, **kw)
        with pytest.raises(ValueError, match=needle):
            SagaDecoder(shape, 2, 16, mode="dense", device="cpu", **kw)


@pytest.mark.parametrize("kw,needle", [
    (dict(mode="atopn", kv_fp8_block=64), "mode 'dense'"), (dict(mode="atopn", kv_budget=8), "mode 'dense'"),
    (dict(mode="vanilla", kv_budget=8), "mode 'dense'"), (dict(kv_budget=8, kv_bits=4), "16- or 8-bit caches"),
    (dict(kv_budget=16), "max_len - 1"), (dict(kv_budget=-1), "max_len - 1"), (dict(kv_budget=8, kv_recent=9), "kv_recent"),
    (dict(kv_budget=8, kv_recent=-1), "kv_recent"), (dict(kv_recent=4), "kv_budget")])
def test_refused_decoders(kw, needle):
    with pytest.raises(ValueError, match=needle):
        SagaDecoder(TINY, 2, 16, **{"mode": "dense", "device": "cpu", **kw})


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("max_len", [1, 64, 65, 300])
def test_8_bit_caches_are_sized_as_built(block, max_len):
    s = replace(TINY, layers=3)
    c = KVCache(s, 2, max_len, "cpu", fp8_block=block)
    assert c.k is None and c.v is None and c.q4 is None
    assert c.nbytes == kv_cache_bytes(s, 2, max_len, fp8_block=block) == sum(t.numel() * t.element_size() for t in c.tensors)
    layer = c.layer(2)
    assert layer.block == block and layer.k_codes.shape == (2, 1, max_len, 64) and layer.v_codes.shape == (2, 2, max_len, 64)
    assert layer.v_scales.shape == (2, 2, -(-max_len // block)) and layer.v_scales.dtype == torch.float32
    assert layer.k_codes.data_ptr() == c.tensors[0][2].data_ptr()
    with pytest.raises(ValueError, match="exclude each other"):
        KVCache(s, 2, max_len, "cpu", bits=4, fp8_block=block)


def test_plans_count_8_bit_caches():
    s, lib = QWEN25_15B_SAGA, _lib.load()
    plan = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X, kv_fp8_block=64)
    wide = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X)
    assert plan.kv_bytes == kv_cache_bytes(s, 8, plan.max_len, fp8_block=64) and plan.total_bytes <= HBM_BYTES_MI355X
    assert 1.9 < plan.max_len / wide.max_len < 2.1
    assert plan.workspace_bytes == decode_workspace_bytes(s, 8, plan.max_len, 512, kv_fp8_block=64)
    for batch in (1, 8):
        rest = [decode_workspace_bytes(s, batch, 4096, 512, **kw) - n for kw, n in (
            (dict(kv_bits=4), lib.saga_dense_q4_workspace_bytes(batch, s.n_q, 4096, s.head_dim)),
            (dict(kv_fp8_block=32), lib.saga_dense_fp8_workspace_bytes(batch, s.n_q, 4096, s.head_dim, 0)))]
        assert rest[0] == rest[1]


def test_a_shape_without_norms_takes_none():
    m = SagaDecoder(TINY, 1, 16, mode="dense", device="cpu", kv_fp8_block=32)
    assert m.q_norm == m.k_norm == [None, None] and m.norm_append and not m.fuse_rope
    m = SagaDecoder(replace(TINY, qk_norm=True), 1, 16, mode="atopn", device="cpu", keep_source_weights=True)
    assert len(m.q_norm) == len(m.k_norm) == 2 and m.q_norm[0].shape == (64,) and m.norm_append
    assert not SagaDecoder(TINY, 1, 16, mode="dense", device="cpu").norm_append
    weights = {n: getattr(m, n) for n in m._WEIGHT_SHAPES}
    del weights["k_norm"]
    with pytest.raises(KeyError, match="k_norm"):
        SagaDecoder(replace(TINY, qk_norm=True), 1, 16, device="cpu", weights=weights)


def test_checkpoints_with_norms(tmp_path):
    pytest.importorskip("transformers")
    from safetensors.torch import load_file, save_file
    from ckpt_util import save_saga_checkpoint, tiny_hf_model
    from saga_amd.checkpoint import load_checkpoint
    path = str(tmp_path / "saga")
    save_saga_checkpoint(tiny_hf_model("llama", n_kv=2, n_k_shared=1, tie=False, d=64), path, n_k=1)
    shape, w = load_checkpoint(path)
    assert not shape.qk_norm and "q_norm" not in w
    sd = load_file(path + "/model.safetensors")
    g = torch.Generator().manual_seed(1)
    for l in range(shape.layers):
        for n in ("q_norm", "k_norm"):
            sd[f"model.layers.{l}.self_attn.{n}.weight"] = torch.rand(64, generator=g) + 0.5
    save_file(sd, path + "/model.safetensors")
    shape, w = load_checkpoint(path)
    assert shape.qk_norm and shape.head_dim == 64
    for l in range(shape.layers):
        for n in ("q_norm", "k_norm"):
            assert torch.equal(w[n][l], sd[f"model.layers.{l}.self_attn.{n}.weight"].to(torch.bfloat16))
    m = SagaDecoder(shape, 1, 16, device="cpu", weights=w)
    assert torch.equal(m.k_norm[1], w["k_norm"][1])
    del sd["model.layers.1.self_attn.k_norm.weight"]
    save_file(sd, path + "/model.safetensors")
    with pytest.raises(KeyError, match="k_norm"):
        load_checkpoint(path)
    sd["model.layers.1.self_attn.k_norm.weight"] = torch.ones(128)  # one norm over two heads is another model
    save_file(sd, path + "/model.safetensors")
    with pytest.raises(ValueError, match="k_norm"):
        load_checkpoint(path)


def test_traces_and_headings_tell_the_cache(monkeypatch, capsys):
    names = set()
    for flags in ([], ["--kv_fp8_block", "64"], ["--kv_fp8_block", "128", "--weight_bits", "4"]):
        seen = []

        def run(cmd, **kw):  # a configuration's subprocess: what it would write and print
            args = speedup.build_parser().parse_args(cmd[3:])
            (mode, param), = speedup.parse_attention(args.attention)
            seen.append(speedup.trace_name("t.json", True, mode, param, 8, 4096, speedup._bits(args)))
            line = '{"mean_ms": 1.5, "std_ms": 0, "p50_ms": 1.4, "p90_ms": 1.6, "tokens_per_s": 5333}'
            return subprocess.CompletedProcess(cmd, 0, stdout=line, stderr="")

        monkeypatch.setattr(speedup.subprocess, "run", run)
        assert speedup.main(["--batch_sizes", "8", "--seq_lengths", "4096", *flags]) == 0
        out = capsys.readouterr().out
        assert ("Caches in 8 bits: a scale per head" in out) == bool(flags)
        assert ("Held in 4 bits: w4" in out) == ("--weight_bits" in flags)
        names.update(seen)
    assert names == {"t_merged_full_bs8_seq4096.json", "t_merged_full_kv8b64_bs8_seq4096.json",
                     "t_merged_full_kv8b128-w4_bs8_seq4096.json"}
    for flags in (["--attention", "atopn:512"], ["--kv_bits", "4"]):
        with pytest.raises(ValueError, match="kv_fp8_block decodes with"):
            speedup.main(["--batch_sizes", "1", "--seq_lengths", "64", "--kv_fp8_block", "64", *flags])


def test_fake_implementation_gives_the_output_shape():
    with FakeTensorMode():
        for b, q_h, k_h, v_h, L, d, block in ((2, 12, 1, 2, 300, 128, 64), (1, 15, 5, 5, 40, 64, 32)):
            q = torch.empty(b, q_h, 1, d, dtype=torch.float16, device="cuda")
            parts = [t for h in (k_h, v_h) for t in (torch.empty(b, h, L, d, dtype=torch.uint8, device="cuda"),
                                                     torch.empty(b, h, -(-L // block), device="cuda"))]
            out = torch.ops.saga.dense_decode_fp8(q, *parts, block)
            assert out.shape == (b, q_h, 1, d) and out.dtype == torch.float16 and out.device.type == "cuda"
    schema = torch.ops.saga.dense_decode_fp8.default._schema
    assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments)
