"""Operators on data held in 4 bits, on the CPU: the weight format, and every refusal before a launch."""
import ctypes

import pytest
import torch

import q4_util as Q
from saga_amd import _lib, ops


def _err():
    return _lib.load().saga_last_error().decode()


def _t(shape, dtype=_lib.DTYPE_BF16, data=0x100000, strides=None):
    d = _lib.SagaTensor()
    d.data, d.dtype, d.ndim = data, dtype, len(shape)
    if strides is None:
        strides, acc = [], 1
        for n in reversed(shape):
            strides.insert(0, acc)
            acc *= n
    for i, (n, s) in enumerate(zip(shape, strides)):
        d.shape[i], d.stride[i] = n, s
    return d


@pytest.mark.parametrize("N,K,group", [(16, 32, 32), (32, 960, 64), (48, 256, 128), (64, 8960, 128)])
def test_quantize_gemv_weight(N, K, group):
    g = torch.Generator().manual_seed(N)
    x = torch.randn(N, K, generator=g) + 2 * torch.randn(N, 1, generator=g)
    x[0] = 0
    x[1] = -0.3
    w = ops.quantize_gemv_weight(x, group)
    assert w.shape == (N, K) and w.codes.shape == (N // 16, (K + 127) // 128, 1024)
    codes, sz = Q.quantise(x, group)
    assert torch.equal(Q.open_weight(w.codes, K), codes)
    assert torch.equal(w.scales.transpose(1, 2).reshape(N, -1), sz)
    s = sz[:, 0::2].repeat_interleave(group, 1).double()
    assert ((Q.weight_values(w) - x.double()).abs() <= s * 0.500001).all()
    assert (Q.weight_values(w)[0] == 0).all()


def test_quantize_refuses():
    for shape, group in (((17, 64), 64), ((16, 96), 64), ((16, 64), 16), ((64,), 64), ((0, 64), 64)):
        with pytest.raises(ValueError, match="4-bit weights need"):
            ops.quantize_gemv_weight(torch.zeros(shape), group)
    for bad in (float("nan"), float("inf"), 1e6):
        x = torch.zeros(16, 64)
        x[3, 5] = bad
        with pytest.raises(ValueError, match="finite"):
            ops.quantize_gemv_weight(x, 64)


def test_cpu_tensors_are_refused():
    w = ops.quantize_gemv_weight(torch.zeros(16, 64), 64)
    cache = Q.random_cache(torch.Generator().manual_seed(0), 1, 1, 1, 4, 64, 32, device="cpu")
    pos = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.gemv_q4(torch.zeros(1, 64, dtype=torch.bfloat16), w), lambda: ops.unpack_gemv_q4([w]),
                 lambda: ops.rope_kv_append_q4(torch.zeros(1, 192), 1, torch.zeros(1, 32, 2), pos, cache),
                 lambda: ops.read_kv_q4(cache, pos), lambda: ops.dense_decode_q4(torch.zeros(1, 1, 1, 64), cache)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def _cache(B=2, n_k=1, n_v=2, L=48, d=128, group=64):
    c = _lib.KvQ4()
    for name, n in (("k", n_k), ("v", n_v)):
        setattr(c, name + "_codes", _t((B, n, L, d // 2), _lib.DTYPE_U8))
        setattr(c, name + "_scales", _t((B, n, L, 2 * d // group), _lib.DTYPE_F16))
    return c


CACHE_ERRORS = [
    (lambda c: setattr(c, "k_codes", _t((2, 1, 48, 64), _lib.DTYPE_F16)), -1, "codes must be u8"),
    (lambda c: setattr(c, "v_scales", _t((2, 2, 48, 4), _lib.DTYPE_BF16)), -1, "scales f16"),
    (lambda c: setattr(c, "k_codes", _t((2, 1, 47, 64), _lib.DTYPE_U8)), -1, "differ"),
    (lambda c: setattr(c, "v_codes", _t((2, 2, 48, 64), _lib.DTYPE_U8, data=0x100004)), -1, "aligned"),
    (lambda c: setattr(c, "k_codes", _t((2, 1, 48, 64), _lib.DTYPE_U8, strides=(4000, 4000, 72, 1))), -1, "multiple of 16"),
    (lambda c: setattr(c, "k_scales", _t((2, 1, 48, 4), _lib.DTYPE_F16, strides=(400, 400, 6, 1))), -1, "aligned to their size"),
    (lambda c: setattr(c, "v_scales", _t((2, 2, 48, 4), _lib.DTYPE_F16, data=0x100004)), -1, "aligned to their size"),
    (lambda c: setattr(c, "v_scales", _t((2, 2, 48, 4), _lib.DTYPE_F16, strides=(400, 400, 8, 2))), -1, "unit innermost"),
    (lambda c: (setattr(c, "v_codes", _t((3, 2, 48, 64), _lib.DTYPE_U8)),
                setattr(c, "v_scales", _t((3, 2, 48, 4), _lib.DTYPE_F16))), -1, "differ in batch"),
    (lambda c: (setattr(c, "k_scales", _t((2, 1, 48, 2), _lib.DTYPE_F16)),
                setattr(c, "v_scales", _t((2, 2, 48, 2), _lib.DTYPE_F16))), -2, "groups of 32 or 64"),
    (lambda c: (setattr(c, "k_codes", _t((2, 1, 48, 48), _lib.DTYPE_U8)),
                setattr(c, "v_codes", _t((2, 2, 48, 48), _lib.DTYPE_U8))), -2, "head_dim"),
    (lambda c: setattr(c, "k_codes", _t((2, 1, 48, 64), _lib.DTYPE_U8, data=0)), -1, "null data"),
    (lambda c: setattr(c, "k_codes", _t((1, 48, 64), _lib.DTYPE_U8)), -1, "4 dims"),
]


@pytest.mark.parametrize("mutate,code,needle", CACHE_ERRORS)
def test_cache_refusals(mutate, code, needle):
    lib, c = _lib.load(), _cache()
    mutate(c)
    q, out = _t((2, 12, 1, 128)), _t((2, 12, 1, 128))
    r = ctypes.byref
    ws = ctypes.c_void_p(0x200000)
    assert lib.saga_dense_decode_q4(r(q), r(c), None, None, 0.1, r(out), ws, 1 << 30, None) == code, _err()
    assert needle in _err()
    assert lib.saga_rope_kv_append_q4(r(_t((2, 15 * 128))), 12, 0x300000, 0x300000, None, r(_t((2, 12, 128))), r(c), None) == code
    assert needle in _err()
    assert lib.saga_kv_q4_read(r(c), 0x300000, None, r(_t((2, 1, 128))), r(_t((2, 2, 128))), None) == code
    assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(q=_t((2, 12, 2, 128))), -2, "l_q == 1"),
    (dict(q=_t((2, 12, 1, 128), _lib.DTYPE_F32)), -2, "bf16 or f16"),
    (dict(q=_t((2, 12, 1, 64))), -1, "differs"),
    (dict(q=_t((3, 12, 1, 128))), -1, "differs"),
    (dict(q=_t((2, 13, 1, 128))), -1, "multiple of v_h"),
    (dict(q=_t((2, 12, 1, 128), data=0x100002)), -1, "16-byte aligned"),
    (dict(out=_t((2, 12, 1, 64))), -1, "out: shape"),
    (dict(mask=_t((2, 1, 1, 47))), -1, "broadcast"),
    (dict(mask=_t((2, 1, 1, 48), _lib.DTYPE_I64)), -1, "mask: dtype"),
    (dict(nbytes=8, cache=_cache(L=4096)), -3, "workspace"),
    (dict(ws=0x200010, cache=_cache(L=4096)), -3, "256-byte"),
    (dict(cache=None), -1, "cache: null"),
])
def test_dense_q4_refusals(change, code, needle):
    a = dict(q=_t((2, 12, 1, 128)), cache=_cache(), mask=None, out=_t((2, 12, 1, 128)), ws=0x200000, nbytes=1 << 30)
    a.update(change)
    r = lambda t: None if t is None else ctypes.byref(t)
    assert _lib.load().saga_dense_decode_q4(r(a["q"]), r(a["cache"]), r(a["mask"]), None, 0.1, r(a["out"]),
                                            ctypes.c_void_p(a["ws"]), a["nbytes"], None) == code, _err()
    assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(qkv=_t((2, 14 * 128))), -1, "row shorter"),
    (dict(qkv=_t((3, 15 * 128)), q_out=_t((3, 12, 128))), -1, "without batch"),
    (dict(q_out=_t((2, 12, 64))), -1, "q_out: shape"),
    (dict(q_out=_t((2, 12, 128), _lib.DTYPE_F16)), -1, "share one float dtype"),
    (dict(qkv=_t((2, 15 * 128), _lib.DTYPE_I32)), -1, "share one float dtype"),
    (dict(table=0), -1, "null"), (dict(pos=0), -1, "null"), (dict(table=0x300008), -1, "aligned"), (dict(n_q=0), -1, "n_q"),
])
def test_append_q4_refusals(change, code, needle):
    a = dict(qkv=_t((2, 15 * 128)), n_q=12, table=0x300000, pos=0x300000, q_out=_t((2, 12, 128)))
    a.update(change)
    assert _lib.load().saga_rope_kv_append_q4(ctypes.byref(a["qkv"]), a["n_q"], a["table"], a["pos"], None,
                                              ctypes.byref(a["q_out"]), ctypes.byref(_cache()), None) == code, _err()
    assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(k=_t((2, 2, 128))), -1, "shapes"), (dict(v=_t((3, 2, 128))), -1, "shapes"),
    (dict(v=_t((2, 2, 128), _lib.DTYPE_F32)), -1, "share one float dtype"), (dict(pos=0), -1, "pos: null"),
    (dict(k=_t((3, 1, 128)), v=_t((3, 2, 128))), -1, "without batch"),
    (dict(k=_t((2, 1, 128), strides=(256, 256, 2))), -1, "innermost"),
])
def test_read_q4_refusals(change, code, needle):
    a = dict(k=_t((2, 1, 128)), v=_t((2, 2, 128)), pos=0x300000)
    a.update(change)
    assert _lib.load().saga_kv_q4_read(ctypes.byref(_cache()), a["pos"], None, ctypes.byref(a["k"]), ctypes.byref(a["v"]),
                                       None) == code, _err()
    assert needle in _err()


def _weight(N=64, K=256, group=64, codes=None, scales=None):
    w = _lib.Q4Weight()
    w.codes = codes or _t((N // 16, (K + 127) // 128, 1024), _lib.DTYPE_U8)
    w.scales = scales or _t((N // 16, K // group, 16, 2), _lib.DTYPE_F16)
    return w


@pytest.mark.parametrize("change,code,needle", [
    (dict(x=_t((33, 256)), y=_t((33, 64))), -2, "32 rows"),
    (dict(x=_t((4, 256), _lib.DTYPE_F16)), -2, "bf16 only"),
    (dict(x=_t((4, 256), data=0x100002)), -1, "16-byte"),
    (dict(y=_t((4, 32))), -1, "y must be"),
    (dict(y=_t((4, 64)), epilogue=2), -1, "y must be"),
    (dict(epilogue=5), -1, "epilogue"),
    (dict(w=_weight(K=384)), -1, "contiguous"),
    (dict(w=_weight(codes=_t((4, 2, 1024), _lib.DTYPE_U8, data=0x100008))), -1, "16-byte"),
    (dict(w=_weight(codes=_t((4, 2, 1024), _lib.DTYPE_BF16))), -1, "u8"),
    (dict(w=_weight(codes=_t((4, 2, 1024), _lib.DTYPE_U8, strides=(4096, 2048, 1)))), -1, "contiguous"),
    (dict(w=_weight(scales=_t((4, 3, 16, 2), _lib.DTYPE_F16))), -1, "multiple of the group"),
    (dict(w=_weight(scales=_t((4, 16, 16, 2), _lib.DTYPE_F16))), -2, "not built"),
    (dict(w=_weight(scales=_t((3, 4, 16, 2), _lib.DTYPE_F16))), -1, "contiguous"),
    (dict(bias=_t((63,))), -1, "bias"), (dict(bias=_t((64,)), epilogue=2, y=_t((4, 32))), -2, "bias with"),
    (dict(w=None), -1, "w: null"),
])
def test_gemv_q4_refusals(change, code, needle):
    a = dict(x=_t((4, 256)), w=_weight(), bias=None, epilogue=0, y=_t((4, 64)))
    a.update(change)
    r = lambda t: None if t is None else ctypes.byref(t)
    assert _lib.load().saga_gemv_q4(r(a["x"]), r(a["w"]), r(a["bias"]), -1.0, a["epilogue"], r(a["y"]), None, 0,
                                    None) == code, _err()
    assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(out=_t((48, 256))), -1, "out must be"), (dict(out=_t((64, 256), _lib.DTYPE_F16)), -2, "bf16 only"),
    (dict(out=_t((64, 256), strides=(260, 1))), -1, "multiple of 16"), (dict(head_rows=3), -1, "head_rows"),
    (dict(head_rows=16, rot=5), -1, "head_rows"), (dict(n=9), -1, "1 to 8"), (dict(n=0), -1, "1 to 8"),
])
def test_unpack_q4_refusals(change, code, needle):
    a = dict(w=_weight(), out=_t((64, 256)), rot=0, head_rows=0, n=1)
    a.update(change)
    item = _lib.UnpackQ4Item(a["w"], a["out"], a["rot"], a["head_rows"])
    assert _lib.load().saga_unpack_gemv_q4(ctypes.byref(item), a["n"], None) == code, _err()
    assert needle in _err()


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.saga_dense_q4_workspace_bytes(8, 12, 33024, 128) > 0
    for bad in ((0, 12, 64, 128), (8, 0, 64, 128), (8, 12, 0, 128), (8, 12, 1 << 31, 128), (1 << 40, 12, 64, 128)):
        assert lib.saga_dense_q4_workspace_bytes(*bad) == 0
    for bad in ((0, 64, 64), (33, 64, 64), (1, 0, 64), (1, 64, 0), (1, 1 << 40, 64), (1, 64, 1 << 40)):
        assert lib.saga_gemv_q4_workspace_bytes(*bad) == 0


def test_decoder_and_planner_options():
    from saga_amd.decoder import QWEN25_15B_SAGA, DecoderShape, SagaDecoder
    from saga_amd.kv_cache import HBM_BYTES_MI355X, KVCache, decode_weight_bytes, kv_cache_bytes, plan_capacity
    s = QWEN25_15B_SAGA
    assert kv_cache_bytes(s, 8, 33024, bits=4, group=64) == 28 * 8 * 3 * 33024 * (64 + 8)
    assert kv_cache_bytes(s, 8, 33024, bits=4, group=32) == 28 * 8 * 3 * 33024 * (64 + 16)
    assert decode_weight_bytes(s, bits=4) < decode_weight_bytes(s) < 2 * decode_weight_bytes(s, bits=4)
    wide = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X)
    q4 = plan_capacity(s, batch=8, budget_bytes=HBM_BYTES_MI355X, kv_bits=4, weight_bits=4)
    assert q4.total_bytes <= HBM_BYTES_MI355X * 0.95
    # 3.556 times by the rows' bytes (256 against 72); what weights and workspaces leave is at most 3 % apart
    assert 3.4 < q4.max_len / wide.max_len < 3.7
    tiny = DecoderShape(2, 64, 4, 1, 2, 64, 128, 256, 1e4, 1e-6)
    c = KVCache(tiny, 3, 16, device="cpu", bits=4, group=32)
    assert c.nbytes == kv_cache_bytes(tiny, 3, 16, bits=4, group=32) and c.k is None
    assert [tuple(t.shape) for t in c.layer(1)] == [(3, 1, 16, 32), (3, 1, 16, 4), (3, 2, 16, 32), (3, 2, 16, 4)]
    with pytest.raises(ValueError, match="groups of 32 or 64"):
        KVCache(tiny, 3, 16, device="cpu", bits=4, group=128)
    with pytest.raises(ValueError, match="16 or 4"):
        KVCache(tiny, 3, 16, device="cpu", bits=8)
    for kw, needle in ((dict(kv_bits=8), "16 or 4"), (dict(kv_bits=4), "mode 'dense'"),
                       (dict(kv_bits=4, mode="dense", dtype=torch.float32), "bf16 or f16"),
                       (dict(weight_bits=4, weight_group=16), "weight_group"),
                       (dict(weight_bits=4, weight_group=128), "multiples of weight_group"),
                       (dict(weight_bits=4, mode="dense", dtype=torch.float16), "needs bf16")):
        with pytest.raises(ValueError, match=needle):
            SagaDecoder(tiny, 2, 32, device="cpu", **kw)


def test_sizes_of_layouts_without_kernels_are_refused():
    from saga_amd.decoder import QWEN25_15B_SAGA, DecoderShape
    from saga_amd.kv_cache import decode_weight_bytes, kv_cache_bytes, plan_capacity
    s, odd = QWEN25_15B_SAGA, DecoderShape(2, 96, 3, 1, 1, 32, 128, 256, 1e4, 1e-6)
    for call in (lambda: kv_cache_bytes(s, 8, 64, bits=4, group=128), lambda: kv_cache_bytes(odd, 8, 64, bits=4, group=32),
                 lambda: plan_capacity(s, batch=8, kv_bits=4, group=128), lambda: decode_weight_bytes(s, bits=4, group=16)):
        with pytest.raises(ValueError, match="groups of 32"):
            call()
    assert plan_capacity(s, batch=8, weight_bits=4, group=128).max_len > 0


def test_command_line_options():
    import argparse
    from saga_amd import speedup
    args = speedup.build_parser().parse_args(["--kv_bits", "4", "--weight_bits", "4"])
    cmd = " ".join(speedup._sub_cmd(args, "full", None, 8, 4096, "merge"))
    assert "--kv_bits 4" in cmd and "--weight_bits 4" in cmd
    plain = " ".join(speedup._sub_cmd(speedup.build_parser().parse_args([]), "full", None, 8, 4096, "merge"))
    assert "bits" not in plain
    with pytest.raises(ValueError, match="full"):
        speedup.main(["--attention", "full,atopn:64", "--kv_bits", "4"])
    assert isinstance(args, argparse.Namespace)
