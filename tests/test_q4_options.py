"""What the planner, the entry points and the command line say about data held in 4 bits (CPU)."""
from dataclasses import replace

import pytest
import torch

from saga_amd import _lib
from saga_amd.decoder import QWEN25_15B_SAGA, SMOLLM2_360M_SAGA, DecoderShape, SagaDecoder
from saga_amd.kv_cache import (HBM_BYTES_MI355X, decode_weight_bytes, decode_workspace_bytes, kv_cache_bytes, plan_capacity,
                               projection_shapes)


def test_plans_are_decoders_that_can_be_built():
    """The same options are refused by the planner and the decoder, and a batch searched for ends at 32 rows."""
    s = QWEN25_15B_SAGA
    plan = plan_capacity(s, max_len=4096, budget_bytes=HBM_BYTES_MI355X, kv_bits=4, weight_bits=4)
    assert plan.batch == 32 and plan.total_bytes <= HBM_BYTES_MI355X * 0.95
    assert plan_capacity(s, max_len=4096, budget_bytes=HBM_BYTES_MI355X, kv_bits=4).batch > 32
    few = plan_capacity(s, max_len=131072, budget_bytes=12 * 10**9, kv_bits=4, weight_bits=4)
    assert 1 < few.batch < 32  # memory ends it first
    tiny = DecoderShape(2, 64, 4, 1, 2, 64, 128, 256, 1e4, 1e-6)
    for shape, batch, kw, needle in (
            (s, 33, dict(weight_bits=4), "at most 32"), (s, 8, dict(weight_bits=4, dtype=torch.float16), "needs bf16"),
            (s, 8, dict(kv_bits=4, dtype=torch.float32), "bf16 or f16"), (s, 8, dict(kv_bits=8), "16 or 4"),
            (s, 8, dict(weight_bits=2), "16 or 4"), (s, 8, dict(kv_bits=4, kv_group=128), "groups of 32 or 64"),
            (s, 8, dict(weight_bits=4, weight_group=16), "groups of 32, 64 or 128"),
            (SMOLLM2_360M_SAGA, 8, dict(weight_bits=4, weight_group=128), "multiples of weight_group"),
            (replace(s, intermediate=8976), 8, dict(weight_bits=4), "multiples of weight_group"),
            (replace(tiny, vocab=250), 8, dict(weight_bits=4), "widths"),
            (replace(tiny, head_dim=32), 8, dict(kv_bits=4), "head dim")):
        with pytest.raises(ValueError, match=needle):
            plan_capacity(shape, batch=batch, budget_bytes=HBM_BYTES_MI355X, **kw)
        small = replace(shape, layers=1, vocab=min(shape.vocab, 256))
        with pytest.raises(ValueError, match=needle):
            SagaDecoder(small, batch, 16, mode="dense", device="cpu", **kw)
    with pytest.raises(ValueError, match="divide every width"):
        decode_weight_bytes(SMOLLM2_360M_SAGA, bits=4, group=128)


def test_plans_size_caches_and_weights_by_their_own_groups():
    s = QWEN25_15B_SAGA
    plan = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X, kv_bits=4, weight_bits=4, kv_group=32, weight_group=128)
    assert plan.kv_bytes == kv_cache_bytes(s, 8, plan.max_len, bits=4, group=32)
    assert plan.weight_bytes == decode_weight_bytes(s, bits=4, group=128) < decode_weight_bytes(s, bits=4, group=32)
    assert plan.workspace_bytes == decode_workspace_bytes(s, 8, plan.max_len, 512, 4, 4)
    both = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X, kv_bits=4, weight_bits=4, group=32)
    assert both.weight_bytes == decode_weight_bytes(s, bits=4, group=32)
    assert both.kv_bytes == kv_cache_bytes(s, 8, both.max_len, bits=4, group=32)


def test_workspaces_of_4_bit_weights_are_the_4_bit_projections():
    """As the decoder allocates it: the largest of its projections'."""
    s, lib = QWEN25_15B_SAGA, _lib.load()
    for batch in (1, 8, 32):
        rest = decode_workspace_bytes(s, batch, 4096, 512) - lib.saga_gemv_workspace_bytes(batch, s.hidden, s.intermediate)
        need = max(lib.saga_gemv_q4_workspace_bytes(batch, n, k) for n, k in projection_shapes(s))
        assert decode_workspace_bytes(s, batch, 4096, 512, weight_bits=4) == rest + need


def _t(shape, dtype, strides):
    d = _lib.SagaTensor()
    d.data, d.dtype, d.ndim = 0x100000, dtype, len(shape)
    for i, (n, s) in enumerate(zip(shape, strides)):
        d.shape[i], d.stride[i] = n, s
    return d


def test_append_refuses_more_tokens_than_a_launch_holds():
    """Four tokens a block of 256 threads, less than 2^32 threads: at most 2^26 - 4 tokens."""
    import ctypes
    cache = _lib.KvQ4(*(_t((2, 1, 48, n), dt, (48 * n, 48 * n, n, 1))
                        for n, dt in ((64, _lib.DTYPE_U8), (4, _lib.DTYPE_F16)) * 2))
    for n in ((1 << 26) - 3, (1 << 26) - 1, 1 << 26):
        qkv, q = _t((n, 3 * 128), _lib.DTYPE_BF16, (0, 1)), _t((n, 1, 128), _lib.DTYPE_BF16, (128, 128, 1))
        assert _lib.load().saga_rope_kv_append_q4(ctypes.byref(qkv), 1, 0x300000, 0x300000, 0x300000, ctypes.byref(q),
                                                  ctypes.byref(cache), None) == -2, n
        assert "sizes too large" in _lib.load().saga_last_error().decode()


def test_traces_and_headings_tell_the_bits(tmp_path, monkeypatch, capsys):
    """A configuration in 4 bits has a trace of its own, and its heading, settings and summary row say so; without
    them the names are the reference's."""
    import subprocess
    from saga_amd import speedup
    assert speedup.trace_name("t.json", True, "full", None, 8, 4096) == "t_merged_full_bs8_seq4096.json"
    names = set()
    for flags in ([], ["--kv_bits", "4"], ["--weight_bits", "4"], ["--kv_bits", "4", "--weight_bits", "4"]):
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
        bits = "-".join(n for n, f in (("kv4", "--kv_bits"), ("w4", "--weight_bits")) if f in flags)
        label = f"full {bits}".strip()
        assert f"### merged / {label} ###" in out and f"merged     {label:<12} 8 " in out
        assert ("Held in 4 bits: " + bits in out) == bool(flags)
        names.update(seen)
    assert len(names) == 4
    assert speedup.trace_name("t.json", False, "atopn", 512, 8, 4096, "w4") == "t_baseline_atopn_512_w4_bs8_seq4096.json"


def test_opening_no_weights_gives_none():
    """As unpack_gemv_weights."""
    from saga_amd import ops
    assert ops.unpack_gemv_weights([]) == [] and ops.unpack_gemv_q4([]) == []
