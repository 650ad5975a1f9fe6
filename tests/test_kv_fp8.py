"""Refusals of the entry points around the 8-bit cache, the norms and the eviction, and the 8-bit form's rule (CPU)."""
import ctypes

import pytest
import torch

import fp8_util as F
from saga_amd import _lib, ops

I64 = 1 << 40


def _err():
    return _lib.load().saga_last_error().decode()


def _t(shape, dtype=_lib.DTYPE_BF16, data=0x100000, strides=None):
    t = _lib.SagaTensor()
    t.data, t.dtype, t.ndim = data, dtype, len(shape)
    acc = 1
    for i in range(len(shape) - 1, -1, -1):
        t.shape[i] = shape[i]
        t.stride[i] = strides[i] if strides else acc
        acc *= shape[i]
    return t


def _cache(B=2, n_k=1, n_v=2, L=48, d=128, block=32, **change):
    nb = (L + block - 1) // block if block > 0 else 1
    parts = dict(k_codes=_t((B, n_k, L, d), _lib.DTYPE_U8), k_scales=_t((B, n_k, nb), _lib.DTYPE_F32),
                 v_codes=_t((B, n_v, L, d), _lib.DTYPE_U8), v_scales=_t((B, n_v, nb), _lib.DTYPE_F32))
    parts.update(change)
    return _lib.KvFp8(*parts.values(), block)


def _r(t):
    return None if t is None else ctypes.byref(t)


CACHE_ERRORS = [
    (dict(block=16), -2, "not built"), (dict(block=0), -2, "not built"), (dict(block=-32), -2, "not built"),
    (dict(d=96), -2, "head_dim"), (dict(d=256), -2, "head_dim"),
    (dict(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_BF16)), -1, "u8"),
    (dict(v_scales=_t((2, 2, 2), _lib.DTYPE_F16)), -1, "f32"),
    (dict(k_scales=_t((2, 1, 3), _lib.DTYPE_F32)), -1, "differ"), (dict(k_scales=_t((2, 2, 2), _lib.DTYPE_F32)), -1, "differ"),
    (dict(k_scales=_t((2, 1, 2), _lib.DTYPE_F32, strides=(4, 4, 2))), -1, "unit innermost"),
    (dict(k_scales=_t((2, 1, 2), _lib.DTYPE_F32, data=0x100002)), -1, "aligned to their type"),
    (dict(v_codes=_t((2, 2, 48, 64), _lib.DTYPE_U8)), -1, "differ in"),
    (dict(v_codes=_t((2, 2, 47, 128), _lib.DTYPE_U8)), -1, "differ in"),
    (dict(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_U8, data=0x100008)), -1, "16-byte"),
    (dict(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_U8, strides=(48 * 128, 48 * 128, 136, 1))), -1, "multiple of 16"),
    (dict(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_U8, strides=(1 << 40, 1 << 40, 1 << 26, 1))), -2, "64 MB"),
    (dict(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_U8, data=0)), -1, "null"),
]


@pytest.mark.parametrize("change,code,needle", CACHE_ERRORS)
def test_cache_refusals(change, code, needle):
    """Every entry point refuses the same caches."""
    lib = _lib.load()
    c = _cache(**change)
    d = c.k_codes.shape[3]
    q, o, w = _t((2, 12, 1, d)), _t((2, 12, 1, d)), _t((2, 1, 48), _lib.DTYPE_F32)
    calls = [
        lambda: lib.saga_dense_decode_fp8(_r(q), _r(c), None, None, 0.1, _r(o), None, 0, 0x200000, 1 << 40, None),
        lambda: lib.saga_norm_rope_kv_append_fp8(_r(_t((2, 15 * d))), 12, 0x300000, None, None, 1e-6, 0x300000, None, 2,
                                                 _r(_t((2, 12, d))), _r(c), None),
        lambda: lib.saga_kv_fp8_read(_r(c), 0x300000, None, _r(_t((2, 1, d))), _r(_t((2, 2, d))), None),
        lambda: lib.saga_evict_kv_fp8(_r(c), _r(w), 0x300000, 10, 2, None, None, 0x300000, 0x200000, 1 << 40, None),
    ]
    for call in calls:
        assert call() == code, _err()
        assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(q=_t((2, 12, 2, 128))), -2, "l_q == 1"), (dict(q=_t((2, 12, 1, 128), _lib.DTYPE_F32)), -2, "bf16 or f16"),
    (dict(q=_t((3, 12, 1, 128)), out=_t((3, 12, 1, 128))), -1, "batch or head dim"),
    (dict(cache=_cache(n_k=5)), -1, "k_h"), (dict(cache=_cache(n_v=5)), -1, "v_h"), (dict(cache=None), -1, "cache: null"),
    (dict(out=_t((2, 12, 1, 64))), -1, "out: shape"), (dict(out=None), -1, "out: null"),
    (dict(mask=_t((2, 1, 1, 47))), -1, "broadcast"), (dict(mask=_t((2, 5, 1, 48))), -1, "broadcast"),
    (dict(mask=_t((2, 1, 1, 48), _lib.DTYPE_I32)), -1, "mask: dtype"),
    (dict(mask=_t((1, 1, 1, 48), strides=(0, 0, 0, 1 << 26))), -2, "2 GB"),
    (dict(mask=_t((2, 1, 1, 48), data=0x100001)), -1, "aligned to its type"),
    (dict(weights=_t((2, 1, 47), _lib.DTYPE_F32)), -1, "weights"), (dict(weights=_t((2, 2, 48), _lib.DTYPE_F32)), -1, "do not divide"),
    (dict(weights=_t((2, 1, 48), _lib.DTYPE_F16)), -1, "weights"), (dict(weights=_t((3, 1, 48), _lib.DTYPE_F32)), -1, "weights"),
    (dict(weights=_t((2, 1, 48), _lib.DTYPE_F32, strides=(0, 0, 1))), -1, "share memory"),
    (dict(weights=_t((2, 1, 48), _lib.DTYPE_F32), nbytes=64), -3, "workspace"),
    (dict(cache=_cache(L=4096), ws=0), -3, "workspace"), (dict(cache=_cache(L=4096), ws=0x200010), -3, "256-byte"),
])
def test_dense_refusals(change, code, needle):
    a = dict(q=_t((2, 12, 1, 128)), cache=_cache(), mask=None, out=_t((2, 12, 1, 128)), weights=None, ws=0x200000, nbytes=1 << 30)
    a.update(change)
    assert _lib.load().saga_dense_decode_fp8(_r(a["q"]), _r(a["cache"]), _r(a["mask"]), None, 0.1, _r(a["out"]), _r(a["weights"]),
                                             1, a["ws"], a["nbytes"], None) == code, _err()
    assert needle in _err()


APPEND_ERRORS = [
    (dict(qkv=_t((2, 14 * 128))), -1, "row shorter"), (dict(q_out=_t((2, 12, 64))), -1, "q_out: shape"),
    (dict(q_out=_t((2, 12, 128), _lib.DTYPE_F16)), -1, "share one float dtype"),
    (dict(qkv=_t((2, 15 * 128), _lib.DTYPE_I32)), -1, "share one float dtype"), (dict(table=0), -1, "rope_table"),
    (dict(table=0x300008), -1, "aligned"), (dict(pos=0), -1, "null"), (dict(n_q=0), -1, "head counts"), (dict(n_q=I64), -2, "too large"),
    (dict(q_norm=_t((64,))), -1, "norms"), (dict(k_norm=_t((128,), _lib.DTYPE_F32)), -1, "norms"),
    (dict(k_norm=_t((128,), strides=(2,))), -1, "norms"), (dict(q_norm=_t((1, 128))), -1, "norm"),
    (dict(q_norm=_t((128,)), eps=-1.0), -1, "eps"), (dict(q_norm=_t((128,)), eps=float("nan")), -1, "eps"),
    (dict(q_out=_t((2, 12, 128), strides=(0, 128, 1))), -1, "share memory"),
    (dict(qkv=_t(((1 << 26) - 3, 15 * 128), strides=(0, 1)), q_out=_t(((1 << 26) - 3, 12, 128))), -2, "too large"),
]


@pytest.mark.parametrize("change,code,needle", APPEND_ERRORS)
@pytest.mark.parametrize("fp8", [False, True])
def test_append_refusals(change, code, needle, fp8):
    a = dict(qkv=_t((2, 15 * 128)), n_q=12, table=0x300000, q_norm=None, k_norm=None, eps=1e-6, pos=0x300000, q_out=_t((2, 12, 128)))
    a.update(change)
    lib, first = _lib.load(), (_r(a["qkv"]), a["n_q"], a["table"], _r(a["q_norm"]), _r(a["k_norm"]), a["eps"], a["pos"])
    if fp8:
        rc = lib.saga_norm_rope_kv_append_fp8(*first, None, 2, _r(a["q_out"]), _r(_cache()), None)
    else:
        rc = lib.saga_norm_rope_kv_append(*first, 0x300000, _r(a["q_out"]), _r(_t((2, 1, 48, 128))), _r(_t((2, 2, 48, 128))), None)
    assert rc == code, _err()
    assert needle in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(v=_t((2, 2, 47, 128))), -1, "shapes"), (dict(v=_t((2, 2, 48, 64))), -1, "shapes"), (dict(k=_t((2, 1, 48, 128), _lib.DTYPE_F16)), -1, "dtype of"),
    (dict(k=_t((2, 1, 48, 96)), v=_t((2, 2, 48, 96))), -2, "not built"), (dict(k=_t((1, 1, 48, 128)), v=_t((1, 2, 48, 128))), -1, "without batch"),
    (dict(k=_t((2, 1, 48, 128), strides=(0, 0, 128, 1))), -1, "share memory"), (dict(k=None), -1, "k_cache: null"),
    (dict(v=_t((2, 2, 48, 128), strides=(48 * 256, 48 * 256, 256, 2))), -1, "innermost"),
])
def test_append_cache_refusals(change, code, needle):
    a = dict(k=_t((2, 1, 48, 128)), v=_t((2, 2, 48, 128)))
    a.update(change)
    assert _lib.load().saga_norm_rope_kv_append(_r(_t((2, 15 * 128))), 12, 0x300000, None, None, 1e-6, 0x300000, None,
                                                _r(_t((2, 12, 128))), _r(a["k"]), _r(a["v"]), None) == code, _err()
    assert needle in _err()


@pytest.mark.parametrize("rows,n,needle", [(0, 2, "rows"), (3, 3, "rows"), (2, 3, "multiple of rows"), (I64, 2, "rows")])
def test_append_rows_refusals(rows, n, needle):
    assert _lib.load().saga_norm_rope_kv_append_fp8(_r(_t((n, 15 * 128))), 12, 0x300000, None, None, 1e-6, 0x300000, None, rows,
                                                    _r(_t((n, 12, 128))), _r(_cache()), None) == -1
    assert needle in _err()
    shared = _cache(k_codes=_t((2, 1, 48, 128), _lib.DTYPE_U8, strides=(0, 0, 128, 1)))
    assert _lib.load().saga_norm_rope_kv_append_fp8(_r(_t((2, 15 * 128))), 12, 0x300000, None, None, 1e-6, 0x300000, None, 2,
                                                    _r(_t((2, 12, 128))), _r(shared), None) == -1 and "share memory" in _err()


@pytest.mark.parametrize("change,code,needle", [
    (dict(k=_t((2, 2, 128))), -1, "shapes"), (dict(v=_t((3, 2, 128))), -1, "shapes"),
    (dict(v=_t((2, 2, 128), _lib.DTYPE_F32)), -1, "share one float dtype"), (dict(pos=0), -1, "pos: null"),
    (dict(k=_t((3, 1, 128)), v=_t((3, 2, 128))), -1, "without batch"), (dict(k=_t((2, 1, 128), strides=(256, 256, 2))), -1, "innermost"),
])
def test_read_refusals(change, code, needle):
    a = dict(k=_t((2, 1, 128)), v=_t((2, 2, 128)), pos=0x300000)
    a.update(change)
    assert _lib.load().saga_kv_fp8_read(_r(_cache()), a["pos"], None, _r(a["k"]), _r(a["v"]), None) == code, _err()
    assert needle in _err()


EVICT_ERRORS = [
    (dict(keep=0), -1, "keep"), (dict(keep=I64), -1, "keep"), (dict(recent=-1), -1, "keep"), (dict(recent=11), -1, "keep"),
    (dict(kv=0), -1, "kv_len"), (dict(kept=0), -1, "kv_len or kept"), (dict(weights=None), -1, "weights: null"),
    (dict(weights=_t((2, 1, 47), _lib.DTYPE_F32)), -1, "weights"), (dict(weights=_t((2, 2, 48), _lib.DTYPE_F32)), -1, "do not divide"),
    (dict(weights=_t((2, 1, 48), _lib.DTYPE_F32, strides=(0, 0, 1))), -1, "share memory"), (dict(nbytes=64), -3, "workspace"),
    (dict(ws=0), -3, "workspace"), (dict(ws=0x200010), -3, "256-byte"),
]


@pytest.mark.parametrize("change,code,needle", EVICT_ERRORS)
@pytest.mark.parametrize("fp8", [False, True])
def test_evict_refusals(change, code, needle, fp8):
    a = dict(weights=_t((2, 1, 48), _lib.DTYPE_F32), kv=0x300000, keep=10, recent=2, kept=0x300000, ws=0x200000, nbytes=1 << 30)
    a.update(change)
    lib, mid = _lib.load(), (_r(a["weights"]), a["kv"], a["keep"], a["recent"])
    if fp8:
        rc = lib.saga_evict_kv_fp8(_r(_cache()), *mid, None, None, a["kept"], a["ws"], a["nbytes"], None)
    else:
        rc = lib.saga_evict_kv(_r(_t((2, 1, 48, 128))), _r(_t((2, 2, 48, 128))), *mid, None, None, None, a["kept"], a["ws"], a["nbytes"], None)
    assert rc == code, _err()
    assert needle in _err()


def test_evict_result_refusals():
    lib = _lib.load()
    w, wo = _t((2, 1, 48), _lib.DTYPE_F32), _t((2, 1, 10), _lib.DTYPE_F32)
    k, v, ko, vo = _t((2, 1, 48, 128)), _t((2, 2, 48, 128)), _t((2, 1, 10, 128)), _t((2, 2, 10, 128))

    def call(k=k, v=v, ko=ko, vo=vo, wo=wo):
        return lib.saga_evict_kv(_r(k), _r(v), _r(w), 0x300000, 10, 2, _r(ko), _r(vo), _r(wo), 0x300000, 0x200000, 1 << 30, None)

    for kw, needle in ((dict(ko=None), "null"), (dict(wo=None), "null"), (dict(ko=_t((2, 1, 9, 128))), "results"),
                       (dict(vo=_t((2, 1, 10, 128))), "results"), (dict(wo=_t((2, 1, 9), _lib.DTYPE_F32)), "weights_out"),
                       (dict(ko=_t((2, 1, 10, 128), _lib.DTYPE_F16)), "one float dtype"),
                       (dict(vo=_t((2, 2, 10, 128), strides=(0, 1280, 128, 1))), "share memory"),
                       (dict(k=_t((2, 1, 48, 96)), v=_t((2, 2, 48, 96)), ko=_t((2, 1, 10, 96)), vo=_t((2, 2, 10, 96))), "not built"),
                       (dict(k=_t((2, 1, 48, 128), data=0x100008)), "16-byte"), (dict(v=_t((2, 2, 47, 128))), "caches")):
        assert call(**kw) < 0 and needle in _err(), (kw, _err())

    def call8(co, wo=wo):
        return lib.saga_evict_kv_fp8(_r(_cache()), _r(w), 0x300000, 10, 2, _r(co), _r(wo), 0x300000, 0x200000, 1 << 30, None)

    for co, needle in ((_cache(L=9), "cache_out"), (_cache(L=10, block=64), "cache_out"), (_cache(L=10, n_v=1), "cache_out"), (None, "cache: null")):
        assert call8(co) == -1 and needle in _err(), _err()
    assert call8(_cache(L=10), None) == -1 and "null" in _err()


def test_evictions_into_their_own_tensors_are_refused():
    """Rows would be overwritten before they are read: in place is the null results' form."""
    lib = _lib.load()
    at = iter(range(1 << 24, 1 << 30, 1 << 24))
    new = lambda shape, dt=_lib.DTYPE_BF16: _t(shape, dt, data=next(at))
    F32, U8 = _lib.DTYPE_F32, _lib.DTYPE_U8
    w, wo, k, v = new((2, 1, 48), F32), new((2, 1, 48), F32), new((2, 1, 48, 128)), new((2, 2, 48, 128))
    ko, vo = new((2, 1, 48, 128)), new((2, 2, 48, 128))
    for kk, vv, ww in ((k, vo, wo), (ko, v, wo), (ko, vo, w), (k, v, w)):
        assert lib.saga_evict_kv(_r(k), _r(v), _r(w), 0x300000, 10, 2, _r(kk), _r(vv), _r(ww), 0x300000, 0x200000, 1 << 30, None) == -1
        assert "must not overlap" in _err()
    parts = lambda: dict(k_codes=new((2, 1, 48, 128), U8), k_scales=new((2, 1, 2), F32), v_codes=new((2, 2, 48, 128), U8),
                         v_scales=new((2, 2, 2), F32))
    src, dst = parts(), parts()
    for name in (*src, None):
        co = _cache(**{**dst, **({name: src[name]} if name else {})})
        rc = lib.saga_evict_kv_fp8(_r(_cache(**src)), _r(w), 0x300000, 10, 2, _r(co), _r(wo if name else w), 0x300000, 0x200000,
                                   1 << 30, None)
        assert rc == -1 and "must not overlap" in _err(), name


def test_appends_refuse_more_rows_than_a_launch_holds():
    """Less than 2^32 threads: blocks of 1024 where 128 positions of 128 dims share a scale."""
    lib = _lib.load()
    for rows, block in (((1 << 21) - 1, 128), ((1 << 23) - 1, 32)):
        qkv, q = _t((rows, 4 * 64 if block == 32 else 4 * 128), strides=(0, 1)), _t((rows, 1, 64 if block == 32 else 128))
        c = _cache(B=rows, L=256, d=64 if block == 32 else 128, block=block)
        assert lib.saga_norm_rope_kv_append_fp8(_r(qkv), 1, 0x300000, None, None, 1e-6, 0x300000, 0x300000, rows, _r(q), _r(c),
                                                None) == -2 and "sizes too large" in _err()


def test_attention_weights_refusals():
    lib = _lib.load()
    q, k, w = _t((2, 12, 1, 128)), _t((2, 2, 48, 128)), _t((2, 2, 48), _lib.DTYPE_F32)

    def call(q=q, k=k, w=w, ws=0x200000, n=1 << 30):
        return lib.saga_attention_weights(_r(q), _r(k), None, None, 0.1, _r(w), 1, ws, n, None)

    for kw, needle in ((dict(w=_t((2, 3, 48), _lib.DTYPE_F32)), "do not divide"), (dict(w=_t((2, 2, 47), _lib.DTYPE_F32)), "weights"),
                       (dict(w=None), "null"), (dict(k=_t((2, 2, 48, 64))), "key"), (dict(q=_t((2, 12, 2, 128))), "l_q"),
                       (dict(ws=0), "workspace"), (dict(ws=0x200008), "256-byte"), (dict(n=64), "workspace")):
        assert call(**kw) < 0 and needle in _err(), (kw, _err())


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.saga_dense_fp8_workspace_bytes(8, 12, 33024, 128, 1) - lib.saga_dense_fp8_workspace_bytes(8, 12, 33024, 128, 0) == 8 * 12 * 33024 * 4
    for bad in ((0, 12, 64, 128, 0), (8, 0, 64, 128, 0), (8, 12, 0, 128, 1), (8, 12, 1 << 31, 128, 0), (1 << 40, 12, 64, 128, 0)):
        assert lib.saga_dense_fp8_workspace_bytes(*bad) == 0
    for bad in ((0, 12, 1, 64), (8, 0, 1, 64), (8, 12, 13, 64), (8, 12, 1, 0), (1 << 40, 12, 1, 64), (1, 12, 1, 1 << 31)):
        assert lib.saga_attention_weights_workspace_bytes(*bad) == 0
    assert lib.saga_evict_workspace_bytes(8, 1, 1000, 10, 3, 256, 1) > lib.saga_evict_workspace_bytes(8, 1, 1000, 10, 3, 256, 0) > 0
    for bad in ((0, 1, 9, 0, 3, 256, 1), (8, 0, 9, 0, 3, 256, 1), (8, 1, 0, 0, 3, 256, 1), (8, 1, 9, 10, 3, 256, 1), (8, 1, 9, -1, 3, 256, 1),
                (8, 1, 9, 0, 0, 256, 1), (8, 1, 9, 0, 3, 0, 1), (8, 1, 1 << 40, 0, 3, 256, 1), (1 << 40, 1, 9, 0, 3, 256, 1)):
        assert lib.saga_evict_workspace_bytes(*bad) == 0


def test_cpu_tensors_are_refused():
    c = ops.KVFP8(torch.zeros(1, 1, 32, 64, dtype=torch.uint8), torch.zeros(1, 1, 1), torch.zeros(1, 1, 32, 64, dtype=torch.uint8),
                  torch.zeros(1, 1, 1), 32)
    x, i, t = torch.zeros(1, 3 * 64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 32, 2)
    k, w = torch.zeros(1, 1, 32, 64), torch.zeros(1, 1, 32)
    for call in (lambda: ops.norm_rope_kv_append(x, 1, t, i, k, k), lambda: ops.norm_rope_kv_append_fp8(x, 1, t, i, c),
                 lambda: ops.read_kv_fp8(c, i), lambda: ops.dense_decode_fp8(k[:, :, :1], c),
                 lambda: ops.attention_weights(k[:, :, :1], k, w), lambda: ops.evict_kv(k, k, w, i, 4), lambda: ops.evict_kv_fp8(c, w, i, 4)):
        with pytest.raises(RuntimeError, match="CPU fallback"):
            call()


# ------------------------------------------------------------------- the rule, as the tests' reference states it

def test_the_reference_form_itself():
    """Rounding against torch's own cast, scales against their definition, blocks that grow."""
    x = torch.cat([torch.randn(4000) * 2.0 ** torch.randint(-12, 8, (4000,)), F.grid().float(), (F.grid()[1:] + F.grid()[:-1]).float() / 2])
    x = x[x.abs() <= 448]
    assert torch.equal(F.nearest(x), x.to(F.F8).view(torch.uint8))
    for top in (1.0, 63.9, 64.0, 1e-20, 3e38, 0.0):
        s = F.scale_of(top)
        assert s == 0.0 if top == 0 else 32 <= top / s < 64
    assert F.scale_of(1e-35) == 2.0 ** -100
    codes, scales = torch.zeros(40, 64, dtype=torch.uint8), torch.zeros(2)
    a, b = torch.randn(20, 64), torch.randn(15, 64) * 100
    F.append(codes, scales, 32, 0, a)
    assert float(scales[0]) == F.scale_of(float(a.abs().max())) and scales[1] == 0
    F.append(codes, scales, 32, 20, b)
    assert float(scales[0]) == F.scale_of(float(b[:12].abs().max())) and float(scales[1]) == F.scale_of(float(b[12:].abs().max()))
    got = F.values(codes[None], scales[None], 32)[0]
    x = torch.cat([a, b]).double()
    # once or, where the scale rose, twice rounded: 2^-4 each of the value, or 2^-10 s
    assert ((got[:35] - x).abs() <= 2 * (2.0 ** -4 * 1.07 * x.abs() + 2.0 ** -10 * float(scales.max()))).all()
    assert F.kept_positions([1.0, 5.0, 0.0, 4.0, 9.0, 2.0], 6, 3, 1) == [4, 1, 5]
    assert F.kept_positions([1.0, 1.0, 1.0], 2, 3, 1) == [0, 1, -1]
