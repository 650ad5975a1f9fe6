"""Attention weights per position and the eviction by them, on the GPU against 64-bit arithmetic and a plain selection."""
import math

import pytest
import torch

import fp8_util as F
from saga_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- weights over a 16-bit cache

def _weights_ref(q, k, mask, kv, scale, G):
    """Sums of softmax weights in 64 bits and a bound: a score's fp32 sums (64 roundings of its largest partial sum, and
    the mask's) move a weight by twice that, the exponential by 2^-20, the sums by L / 16 + 64 roundings."""
    b, q_h, _, _ = q.shape
    L = k.shape[2]
    w, tol = (torch.zeros(b, G, L, dtype=torch.float64, device="cuda") for _ in range(2))
    for i in range(b):
        n = L if kv is None else min(max(int(kv[i]), 0), L)
        for h in range(q_h):
            kd, qd = k[i, h * k.shape[1] // q_h, :n].double(), q[i, h, 0].double()
            x, e = kd @ qd * scale, kd.abs() @ qd.abs() * scale * 64 * U32
            if mask is not None:
                m = mask[i % mask.shape[0], h % mask.shape[1], 0, :n].double()
                x, e = x + m, e + torch.where(m.isfinite(), m.abs(), torch.zeros_like(m)) * U32
            p = torch.softmax(x, 0).nan_to_num(0.0)
            w[i, h * G // q_h, :n] += p
            if n:
                tol[i, h * G // q_h, :n] += p * (2 * (2 * float(e.max()) + 2.0 ** -20) + (n / 16 + 64 + q_h) * U32)
    return w, tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("q_h,k_h,d,G", [(12, 1, 128, 1), (15, 5, 64, 5), (12, 4, 64, 2), (16, 1, 128, 1), (6, 6, 128, 1)])
@pytest.mark.parametrize("L", [1, 33, 1023, 5000])
def test_attention_weights(q_h, k_h, d, G, L, dtype):
    g = _gen(q_h + L)
    b = 3
    q, k = _randn(g, b, q_h, 1, d, dtype=dtype), _randn(g, b, k_h, L, d, dtype=dtype)
    kv = _int32([L, 0, max(1, L // 3)])
    mask = torch.zeros(b, 1, 1, L + 2, device="cuda")
    mask[0, ..., ::3] = float("-inf") if L > 1 else 0.0
    for m in (None, mask):
        ref, tol = _weights_ref(q, k, m if m is None else m[..., :L], kv, 0.1, G)
        w = torch.full((b, G, L), float("nan"), device="cuda")
        assert ops.attention_weights(q, k, w, attention_mask=m, scaling=0.1, kv_len=kv, add=False) is w
        assert ((w.double() - ref).abs() <= tol).all() and not w[1].any()
        more = torch.rand(b, G, L + 3, generator=g, device="cuda")
        want = more.clone()
        want[..., :L] += w
        ops.attention_weights(q, k, more, attention_mask=m, scaling=0.1, kv_len=kv)
        assert torch.equal(more, want)


def test_attention_weights_many_positions():
    """Rows of several thousand positions in many batch rows: blocks of 1024 positions."""
    g = _gen(3)
    q, k = _randn(g, 40, 12, 1, 64, dtype=torch.bfloat16), _randn(g, 40, 2, 9001, 64, dtype=torch.bfloat16)
    kv = _int32([9001 - 200 * i for i in range(40)])
    ref, tol = _weights_ref(q, k, None, kv, 0.125, 2)
    w = torch.empty(40, 2, 9001, device="cuda")
    ops.attention_weights(q, k, w, kv_len=kv, add=False)
    assert ((w.double() - ref).abs() <= tol).all()
    assert torch.equal(w, ops.attention_weights(q, k, torch.empty_like(w), kv_len=kv, add=False))  # no order that changes


def test_attention_weights_of_several_queries():
    """The last queries of a prompt as rows of an expanded key, each with its own length."""
    g = _gen(4)
    L, n, d = 500, 7, 128
    k, q = _randn(g, 1, 2, L, d, dtype=torch.bfloat16), _randn(g, n, 4, 1, d, dtype=torch.bfloat16)
    kv = torch.arange(L - n + 1, L + 1, device="cuda").int()
    wide = k.expand(n, -1, -1, -1)
    ref, tol = _weights_ref(q, wide, None, kv, 0.1, 2)
    w = ops.attention_weights(q, wide, torch.empty(n, 2, L, device="cuda"), scaling=0.1, kv_len=kv, add=False)
    assert ((w.double() - ref).abs() <= tol).all()


def test_attention_weights_nan_and_refusals():
    g = _gen(5)
    q, k = _randn(g, 2, 4, 1, 64, dtype=torch.float16), _randn(g, 2, 2, 100, 64, dtype=torch.float16)
    k[1, 0, 50, 3] = float("nan")
    w = ops.attention_weights(q, k, torch.zeros(2, 2, 100, device="cuda"))
    assert w.isfinite().all() and not w[1, 0].any() and abs(float(w[1, 1].sum()) - 2) < 1e-5
    for bad, needle in ((torch.zeros(2, 3, 100, device="cuda"), "do not divide"), (torch.zeros(2, 2, 99, device="cuda"), "f32"),
                        (torch.zeros(2, 2, 100, device="cuda", dtype=torch.float16), "f32"),
                        (torch.zeros(1, 2, 100, device="cuda").expand(2, -1, -1), "share memory")):
        with pytest.raises(RuntimeError, match=needle):
            ops.attention_weights(q, k, bad)


# ------------------------------------------------------------------- eviction

def _random_weights(g, kind, b, G, L):
    w = torch.exp(3 * _randn(g, b, G, L))
    if kind == "ties":
        w = torch.randint(0, 4, (b, G, L), generator=g, device="cuda").float()
        w = torch.where(torch.rand(b, G, L, generator=g, device="cuda") < 0.1, -0.0 * w, w)
    elif kind == "zeros":
        w = w * (torch.rand(b, G, L, generator=g, device="cuda") < 0.05)
    elif kind == "special":
        r = torch.rand(b, G, L, generator=g, device="cuda")
        w = torch.where(r < 0.02, torch.full_like(w, float("nan")), w)
        w = torch.where((r > 0.02) & (r < 0.04), torch.full_like(w, float("inf")), w)
        w = torch.where((r > 0.04) & (r < 0.1), -w, w)
        w = torch.where((r > 0.1) & (r < 0.12), torch.full_like(w, float("-inf")), w)
        w = torch.where((r > 0.12) & (r < 0.13), torch.full_like(w, -float("nan")), w)
    elif kind == "same":
        w = torch.full_like(w, 0.25)
    elif kind == "rising":
        w = torch.arange(L, device="cuda").float().expand(b, G, L).contiguous()
    elif kind == "falling":
        w = -torch.arange(L, device="cuda").float().expand(b, G, L).contiguous()
    return w


def _check_evict(w, kv, keep, recent, k, v, block=None):
    """Both forms, rows of k and v (16 bits, or a KVFP8 in k) against the plain selection."""
    b, G, L = w.shape
    lens = [min(max(int(n), 0), L) for n in kv]
    rows = w.cpu().tolist()
    want = torch.tensor([[F.kept_positions(r, lens[i], keep, recent) for r in rows[i]] for i in range(b)], device="cuda")
    tensors = list(k[:4]) if block else [k, v]
    heads = [t.shape[1] for t in ((k.k_codes, k.v_codes) if block else tensors)]
    live = want >= 0

    def moved(t, h):  # rows of t [b, h, L, ...] at the kept positions
        at = want.clamp(min=0).repeat_interleave(h // G, 1)
        return t.gather(2, at.reshape(*at.shape, *[1] * (t.dim() - 3)).expand(*at.shape, *t.shape[3:]))

    ww = w.gather(-1, want.clamp(min=0))
    if block:
        nb = -(-keep // block)
        expect = []
        for codes, scales, h in ((k.k_codes, k.k_scales, heads[0]), (k.v_codes, k.v_scales, heads[1])):
            there = live.repeat_interleave(h // G, 1)
            s = scales.gather(-1, want.clamp(min=0).repeat_interleave(h // G, 1) // block).double() * there
            top = torch.nn.functional.pad(s, (0, nb * block - keep)).unflatten(-1, (nb, block)).amax(-1)
            by = top.repeat_interleave(block, -1)[..., :keep]
            r = torch.where(by > 0, s / torch.where(by > 0, by, torch.ones_like(by)), torch.ones_like(by))
            c = F.nearest(F.opened(moved(codes, h)) * r[..., None])
            expect.append((torch.where((r == 1)[..., None], moved(codes, h), c), top.float(), there))
        out = ops.KVFP8(*(torch.full((b, h, m, *t), f, dtype=dt, device="cuda") for h in heads for m, t, f, dt in
                          ((keep + 3, (k.k_codes.shape[-1],), 0x55, torch.uint8), (-(-(keep + 3) // block), (), 9.0, torch.float32))), block)
        w_out = torch.full((b, G, keep + 5), 3.0, device="cuda")
        before = F.clone(k)
        kept = ops.evict_kv_fp8(k, w, kv, keep, recent, out=(out, w_out))
        assert F.same(k, before)
        for (codes, top, there), got_c, got_s in zip(expect, (out.k_codes, out.v_codes), (out.k_scales, out.v_scales)):
            assert torch.equal(F.bits(got_c[:, :, :keep]), F.bits(torch.where(there[..., None], codes, torch.full_like(codes, 0x55))))
            assert (got_c[:, :, keep:] == 0x55).all()
            some = torch.nn.functional.pad(there, (0, nb * block - keep)).unflatten(-1, (nb, block)).any(-1)
            assert torch.equal(got_s[..., :nb], torch.where(some, top, torch.full_like(top, 9.0)))
    else:
        out = [torch.full((b, t.shape[1], keep + 3, t.shape[-1]), 5.0, dtype=t.dtype, device="cuda") for t in tensors]
        w_out = torch.full((b, G, keep + 5), 3.0, device="cuda")
        before = [t.clone() for t in tensors]
        kept = ops.evict_kv(k, v, w, kv, keep, recent, out=(*out, w_out))
        assert all(torch.equal(a, c) for a, c in zip(tensors, before))
        for t, got in zip(tensors, out):
            there = live.repeat_interleave(t.shape[1] // G, 1)[..., None]
            assert torch.equal(got[:, :, :keep], torch.where(there, moved(t, t.shape[1]), torch.full_like(got[:, :, :keep], 5.0)))
            assert (got[:, :, keep:] == 5).all()
    assert torch.equal(kept.long(), want)
    bits = lambda t: t.contiguous().view(torch.int32)
    assert torch.equal(bits(w_out[..., :keep]), bits(torch.where(live, ww, torch.zeros_like(ww)))) and not w_out[..., keep:].any()
    # in place: the same places, what lies behind is left, weights there are 0
    w2 = w.clone()
    place = torch.arange(L, device="cuda")
    cut = torch.tensor([min(n, keep) for n in lens], device="cuda")[:, None, None]
    if block:
        mine = F.clone(k)
        kept2 = ops.evict_kv_fp8(mine, w2, kv, keep, recent)
        for i, h in ((0, heads[0]), (2, heads[1])):
            m = min(keep, L)
            there = live[..., :m].repeat_interleave(h // G, 1)[..., None]
            assert torch.equal(F.bits(mine[i][:, :, :m]), F.bits(torch.where(there, expect[i // 2][0][:, :, :m], k[i][:, :, :m])))
            assert torch.equal(mine[i][:, :, m:], k[i][:, :, m:])
            some = there[..., 0].clone()
            some = torch.nn.functional.pad(some, (0, -m % block)).unflatten(-1, (-1, block)).any(-1)
            n2 = some.shape[-1]
            assert torch.equal(mine[i + 1][..., :n2], torch.where(some, expect[i // 2][1][..., :n2], k[i + 1][..., :n2]))
            assert torch.equal(mine[i + 1][..., n2:], k[i + 1][..., n2:])
    else:
        mine = [t.clone() for t in tensors]
        kept2 = ops.evict_kv(*mine, w2, kv, keep, recent)
        for t, got in zip(tensors, mine):
            m = min(keep, L)
            there = live[..., :m].repeat_interleave(t.shape[1] // G, 1)[..., None]
            assert torch.equal(got[:, :, :m], torch.where(there, moved(t, t.shape[1])[:, :, :m], t[:, :, :m]))
            assert torch.equal(got[:, :, m:], t[:, :, m:])
    assert torch.equal(kept, kept2)
    full = torch.nn.functional.pad(ww, (0, max(L - keep, 0)))[..., :L]
    assert torch.equal(bits(w2), bits(torch.where(place < cut, full, torch.zeros_like(full))))


KINDS = ["random", "ties", "zeros", "special", "same", "rising", "falling"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("keep,recent", [(100, 20), (100, 0), (100, 100), (1, 0), (1, 1), (299, 1), (64, 32), (300, 7), (500, 200)])
def test_evict_selection(kind, keep, recent):
    """Weights of every kind; rows longer than, as long as and shorter than what is kept, empty ones."""
    g = _gen(keep + recent)
    b, G, L, d = 5, 2, 300, 64
    w = _random_weights(g, kind, b, G, L)
    kv = _int32([300, keep if keep < 300 else 299, 0, min(keep + 1, 300), -2])
    k, v = _randn(g, b, 2, L, d, dtype=torch.bfloat16), _randn(g, b, 4, L, d, dtype=torch.bfloat16)
    _check_evict(w, kv, keep, recent, k, v)
    _check_evict(w, kv, keep, recent, F.random_cache(g, b, 2, 4, L, d, 32), None, 32)


@pytest.mark.parametrize("L", [8192, 8193, 33000, 65536, 65537, 150001])
@pytest.mark.parametrize("kind", ["random", "zeros", "special"])
def test_evict_long_rows(L, kind):
    """Lengths around what a selection holds at a time (32768 positions), and several of it."""
    g = _gen(L)
    w = _random_weights(g, kind, 2, 1, L)
    k, v = _randn(g, 2, 1, L, 64, dtype=torch.float16), _randn(g, 2, 1, L, 64, dtype=torch.float16)
    _check_evict(w, _int32([L, L - 1000]), L // 2 + 1, 513, k, v)


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("d,k_h,v_h,G", [(128, 1, 2, 1), (64, 5, 5, 5), (64, 2, 6, 1), (128, 3, 3, 3)])
def test_evict_layouts(block, d, k_h, v_h, G):
    """Blocks of scales of very different sizes; in place the staged end begins inside a block; types of rows."""
    g = _gen(block + d + k_h)
    b, L = 3, 1000
    cache = F.random_cache(g, b, k_h, v_h, L, d, block)
    for s in (cache.k_scales, cache.v_scales):
        s *= torch.exp2(torch.randint(-9, 9, s.shape, generator=g, device="cuda").float())
        s[0, 0, :2] = 0.0
    cache.k_codes[:, 0, 7, 3], cache.v_codes[:, -1, 900, 5] = 0x7f, 0xff
    w = _random_weights(g, "random", b, G, L)
    w[:, :, 7] = 1e9  # (the NaN among the kept)
    kv = _int32([1000, 777, 400])
    for keep, recent in ((500, 90), (501, 333), (128, 128), (700, 0), (65, 1)):
        _check_evict(w, kv, keep, recent, cache, None, block)
    for dtype in (torch.float32, torch.float16):
        k, v = _randn(g, b, k_h, L, d, dtype=dtype), _randn(g, b, v_h, L, d, dtype=dtype)
        _check_evict(w, kv, 501, 77, k, v)


def test_evict_views():
    """Strided caches and weights, a batch row of a larger cache, a caller's kept and workspace."""
    g = _gen(9)
    b, L, d = 2, 300, 64
    k, v = (_randn(g, b, L, 3, d + 8, dtype=torch.bfloat16).transpose(1, 2)[:, :h, :, :d] for h in (1, 3))
    w = _randn(g, b, 3, L + 7).abs()[:, ::3, :L]
    kv = _int32([300, 250])
    kc, vc, wc = k.contiguous(), v.contiguous(), w.contiguous()
    want = ops.evict_kv(kc, vc, wc, kv, 100, 30)
    kept = torch.empty(b, 1, 100, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert ops.evict_kv(k, v, w, kv, 100, 30, kept=kept, workspace=ws) is kept
    assert torch.equal(kept, want) and torch.equal(k, kc) and torch.equal(v, vc) and torch.equal(w, wc)
    cache = F.random_cache(g, 3, 1, 1, L, d, 32)
    w = _randn(g, 3, 1, L).abs()
    alone = ops.KVFP8(*(t[1:2].clone() for t in cache[:4]), 32)
    others = F.clone(cache)
    ops.evict_kv_fp8(alone, w[1:2].clone(), kv[:1], 99, 9)
    ops.evict_kv_fp8(cache.rows(1), w[1:2], kv[:1], 99, 9)
    assert F.same(cache.rows(1), alone) and F.same(cache.rows(0), others.rows(0)) and F.same(cache.rows(2), others.rows(2))


def test_evict_refusals():
    g = _gen(10)
    k, v, w, kv = (_randn(g, 2, 2, 50, 64), _randn(g, 2, 3, 50, 64), _randn(g, 2, 1, 50), _int32([50, 50]))
    for bad in ((0, 0), (10, 11), (10, -1)):
        with pytest.raises(ValueError, match="keep"):
            ops.evict_kv(k, v, w, kv, *bad)
    with pytest.raises(ValueError, match="kv_len"):
        ops.evict_kv(k, v, w, kv[:1], 10)
    with pytest.raises(ValueError, match="kv_len"):
        ops.evict_kv(k, v, w, None, 10)
    with pytest.raises(RuntimeError, match="do not divide"):
        ops.evict_kv(k, v, _randn(g, 2, 2, 50), kv, 10)
    with pytest.raises(ValueError, match="kept"):
        ops.evict_kv(k, v, w, kv, 10, kept=torch.empty(2, 1, 9, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="results"):
        ops.evict_kv(k, v, w, kv, 10, out=(k[:, :, :9].clone(), v.clone(), w.clone()))
    with pytest.raises(RuntimeError, match="share memory"):
        ops.evict_kv(k[:1].expand(2, -1, -1, -1), v, w, kv, 10)
    with pytest.raises(RuntimeError, match="null"):
        ops.evict_kv(k, v, w, kv, 10, out=(k.clone(), v.clone(), None))


@pytest.mark.parametrize("fp8", [False, True])
def test_bounded_decode_captured_and_replayed(fp8):
    """Steps in a cache of 96 places that is cut to 40 whenever it is full, step and eviction as two graphs: each equals
    the eager calls, and at every step the attention is that over the kept positions' rows."""
    g = _gen(11 + fp8)
    B, L, n_q, n_k, n_v, d, block, keep, recent = 3, 96, 6, 1, 2, 64, 32, 40, 11

    def state():
        if fp8:
            c = ops.KVFP8(*(torch.zeros(s, dtype=t, device="cuda") for h in (n_k, n_v) for s, t in
                            (((B, h, L, d), torch.uint8), ((B, h, 3), torch.float32))), block)
        else:
            c = [torch.zeros(B, h, L, d, dtype=torch.bfloat16, device="cuda") for h in (n_k, n_v)]
        return dict(c=c, w=torch.zeros(B, 1, L, device="cuda"), slot=_int32([0] * B), kv=_int32([0] * B))

    qkv, pos = _randn(g, B, 9 * d, dtype=torch.bfloat16), _int32([0] * B)
    one = torch.ones(d, dtype=torch.bfloat16, device="cuda")

    def step(s):
        table = ops.rope_table(pos, d, 1e4)
        s["kv"] += 1
        if fp8:
            q = ops.norm_rope_kv_append_fp8(qkv, n_q, table, s["slot"], s["c"], one, one).view(B, n_q, 1, d)
            s["out"] = ops.dense_decode_fp8(q, s["c"], kv_len=s["kv"], weights=s["w"])
        else:
            q = ops.norm_rope_kv_append(qkv, n_q, table, s["slot"], *s["c"], one, one).view(B, n_q, 1, d)
            s["out"] = ops.dense_decode(q, *s["c"], kv_len=s["kv"])
            ops.attention_weights(q, s["c"][0], s["w"], kv_len=s["kv"])
        s["slot"] += 1

    def cut(s):
        if fp8:
            s["kept"] = ops.evict_kv_fp8(s["c"], s["w"], s["kv"], keep, recent)
        else:
            s["kept"] = ops.evict_kv(*s["c"], s["w"], s["kv"], keep, recent)
        s["kv"].clamp_(max=keep)
        s["slot"].clamp_(max=keep)

    a, e = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a)
        cut(a)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (step, cut):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            f(a)
        graphs.append(graph)
    for t in (*a["c"][:4], a["w"], a["slot"], a["kv"]):
        t.zero_()
    held = [[] for _ in range(B)]  # the positions that the places hold
    for i in range(250):
        qkv.copy_(_randn(g, B, 9 * d, dtype=torch.bfloat16))
        pos.fill_(i)
        if int(e["kv"][0]) == L:
            graphs[1].replay()
            kept = a["kept"].clone()
            cut(e)
            assert torch.equal(kept, e["kept"])
            for r in range(B):
                held[r] = [held[r][j] for j in kept[r, 0].tolist()]
                assert held[r][-recent:] == list(range(i - recent, i))
        graphs[0].replay()
        got = a["out"].clone()
        step(e)
        assert torch.equal(got, e["out"]), i
        assert got.isfinite().all()
        for r in range(B):
            held[r].append(i)
    for x, y in zip(a["c"][:4], e["c"][:4]):
        assert torch.equal(x, y)
    assert torch.equal(a["w"], e["w"]) and int(e["kv"][0]) < L and len(held[0]) == int(e["kv"][0])
    ops.clear_workspaces()


@pytest.mark.parametrize("fp8", [False, True])
def test_two_rows_past_32_bit_offsets(fp8):
    """Rows whose byte offsets pass 2^32: the last positions are kept and read."""
    g = _gen(12)
    L, d = (1 << 25) + 320, 128
    n = 300
    w = torch.zeros(1, 1, L, device="cuda")
    w[..., : n // 2] = 1.0
    if fp8:
        codes = torch.zeros(1, 1, L, d, dtype=torch.uint8, device="cuda")
        codes[:, :, -n:] = torch.randint(0, 100, (1, 1, n, d), generator=g, device="cuda").to(torch.uint8)
        cache = ops.KVFP8(codes, torch.ones(1, 1, L // 32, device="cuda"), codes, torch.ones(1, 1, L // 32, device="cuda"), 32)
        out = ops.KVFP8(*(t.clone() for t in (codes[:, :, :512], cache.k_scales[..., :16]) * 2), 32)
        kept = ops.evict_kv_fp8(cache, w, _int32([L]), 450, 300, out=(out, torch.zeros(1, 1, 450, device="cuda")))
        assert torch.equal(out.k_codes[:, :, 150:450], codes[:, :, -n:]) and torch.equal(out.v_codes, out.k_codes)
    else:
        k = torch.zeros(1, 1, L, d, dtype=torch.bfloat16, device="cuda")
        k[:, :, -n:] = _randn(g, 1, 1, n, d, dtype=torch.bfloat16)
        rows = k[:, :, -n:].clone()
        kept = ops.evict_kv(k, torch.zeros(1, 1, L, d, dtype=torch.bfloat16, device="cuda"), w, _int32([L]), 450, 300)
        assert torch.equal(k[:, :, 150:450], rows)
    assert kept[0, 0, :150].tolist() == list(range(150)) and kept[0, 0, 150:].tolist() == list(range(L - n, L))
