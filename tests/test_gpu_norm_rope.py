"""Norms of queries and keys with the rotation and the append in one pass, into caches of the tokens' own type."""
import pytest
import torch

from saga_amd import ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}
# Below its smallest normal number a type's numbers are evenly spaced (f16: 2^-24 under 2^-14): half a step there.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def _reference(qkv, table, n_q, n_k, d, q_norm, k_norm, eps):
    """Queries, keys, values in 64 bits and a bound of the fp32 error: the sum of d / 16 * 16 squares has 16 + 3 additions
    and as many products, the root, the quotient and two more products follow, and a rotation's two products and their
    sum: less than 24 roundings, each of half a step of |a cos| + |b sin|."""
    x = qkv.double().reshape(qkv.shape[0], -1, d)
    cs, sn = table[:, None, :, 0].double(), table[:, None, :, 1].double()
    outs = []
    for t, w in ((x[:, :n_q], q_norm), (x[:, n_q:n_q + n_k], k_norm)):
        if w is not None:
            t = t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        a, b = t[..., : d // 2], t[..., d // 2:]
        size = torch.cat([(a * cs).abs() + (b * sn).abs(), (b * cs).abs() + (a * sn).abs()], -1)
        outs += [torch.cat([a * cs - b * sn, b * cs + a * sn], -1), 24 * U32 * size]
    return outs, x[:, n_q + n_k:]


def _close(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_q,n_k,n_v,d", [(12, 1, 2, 128), (15, 1, 5, 64), (4, 2, 2, 128), (5, 5, 1, 64), (1, 1, 1, 64)])
@pytest.mark.parametrize("n", [1, 7, 333, 1500])
def test_norm_rope_append(n, n_q, n_k, n_v, d, dtype):
    """Queries, cache rows and nothing else, with both norms, one and none; rows apart from the rotations' positions."""
    g = _gen(n + d + n_q)
    B, L = 3, 700
    qkv = _randn(g, n, (n_q + n_k + n_v) * d)
    qkv.view(n, -1, d)[:, :, ::7] += 3.0
    qkv = qkv.to(dtype)
    at = torch.randperm(B * L, generator=g, device="cuda")[:n]
    pos, batch = (at % L).int(), (at // L).int()
    table = ops.rope_table((torch.arange(n, device="cuda") * 37).int(), d, 1e4)
    qn, kn = (1 + 0.3 * _randn(g, d)).to(dtype), (0.5 + 0.3 * _randn(g, d)).to(dtype)
    for norms in ((qn, kn), (None, kn), (qn, None), (None, None)):
        kc, vc = (_randn(g, B, h, L, d, dtype=dtype) for h in (n_k, n_v))
        k0, v0 = kc.clone(), vc.clone()
        q = ops.norm_rope_kv_append(qkv, n_q, table, pos, kc, vc, *norms, eps=1e-5, batch=batch)
        (qr, qt, kr, kt), v = _reference(qkv, table, n_q, n_k, d, *norms, 1e-5)
        _close(q, qr, qt + HALF[dtype] * (qr.abs() + qt) + TINY[dtype])
        _close(kc[batch.long(), :, pos.long()], kr, kt + HALF[dtype] * (kr.abs() + kt) + TINY[dtype])
        assert torch.equal(vc[batch.long(), :, pos.long()].double(), v)
        k0[batch.long(), :, pos.long()], v0[batch.long(), :, pos.long()] = kc[batch.long(), :, pos.long()], vc[batch.long(), :, pos.long()]
        assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_without_norms_as_rope_kv_append():
    """No norms and the same rotations: the bits of rope_kv_append."""
    g, n, n_q, n_k, n_v, d, B, L = _gen(2), 9, 12, 1, 2, 128, 9, 64
    qkv = _randn(g, n, 15 * d, dtype=torch.bfloat16)
    pos = torch.randint(0, L, (n,), generator=g, device="cuda").int()
    a, b = ([torch.zeros(B, h, L, d, dtype=torch.bfloat16, device="cuda") for h in (n_k, n_v)] for _ in range(2))
    q = ops.rope_kv_append(qkv, n_q, n_k, n_v, 1e6, pos, *a)
    q2 = ops.norm_rope_kv_append(qkv, n_q, ops.rope_table(pos, d, 1e6), pos, *b)
    assert torch.equal(q, q2) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_special_values_and_out_of_range():
    """A zero head stays zero (eps), a NaN or an infinity reaches its own head, an index out of range no cache row."""
    g, n_q, n_k, n_v, d, B, L = _gen(3), 2, 1, 1, 64, 2, 16
    qkv = _randn(g, 6, 4 * d)
    x = qkv.view(6, 4, d)
    x[0, 0] = 0.0
    x[1, 2, 5], x[2, 3, 7], x[5, 0, 1] = float("nan"), float("inf"), float("inf")
    x[4] *= 1e-20  # squares below fp32: the norm leaves x / sqrt(eps)
    pos = torch.tensor([0, 15, 3, -1, 16, 4], dtype=torch.int32, device="cuda")
    batch = torch.tensor([0, 1, 1, 0, 0, 1], dtype=torch.int32, device="cuda")
    table = ops.rope_table(pos.clamp(min=0), d, 1e4)
    kc, vc = (torch.full((B, 1, L, d), 7.0, device="cuda") for _ in range(2))
    one = torch.ones(d, device="cuda")
    q = ops.norm_rope_kv_append(qkv, n_q, table, pos, kc, vc, one, one, batch=batch)
    assert q[[3, 4]].isnan().all() and (q[0, 0] == 0).all() and q[[0, 1, 2]].isfinite().all()
    assert q[5, 0].isnan().any() and q[5, 1].isfinite().all()
    assert kc[1, 0, 15].isnan().all() and kc[0, 0, 0].isfinite().all() and vc[1, 0, 3, 7] == float("inf")
    written = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    written[[0, 1, 1, 1], [0, 15, 3, 4]] = True
    assert (kc[:, 0][~written] == 7).all() and (vc[:, 0][~written] == 7).all()
    assert ops.norm_rope_kv_append(qkv[:2], n_q, table[:2].contiguous(), pos[:2].contiguous(), kc, vc, eps=0.0).isfinite().all()


def test_views_and_unaligned_rows():
    """Projections, queries, norms and caches that start or step off 16 bytes give what aligned ones do."""
    g, n, n_q, n_k, n_v, d, B, L = _gen(4), 5, 4, 1, 2, 128, 5, 32
    qkv = _randn(g, n, 7 * d, dtype=torch.float16)
    wide = torch.zeros(n, 7 * d + 3, dtype=torch.float16, device="cuda")
    wide[:, 1:-2] = qkv
    pos = torch.randint(0, L, (n,), generator=g, device="cuda").int()
    table = ops.rope_table(pos, d, 1e4)
    norm = (1 + _randn(g, d + 1) * 0.1).half()
    kc, vc = (torch.zeros(B, h, L, d, dtype=torch.float16, device="cuda") for h in (n_k, n_v))
    odd = [torch.zeros(B, L, h, d + 1, dtype=torch.float16, device="cuda").transpose(1, 2)[..., 1:] for h in (n_k, n_v)]
    q = ops.norm_rope_kv_append(qkv, n_q, table, pos, kc, vc, norm[1:].clone(), norm[1:].clone())
    q2 = torch.zeros(n, d + 5, n_q, dtype=torch.float16, device="cuda").transpose(1, 2).contiguous()[..., 5:]
    ops.norm_rope_kv_append(wide[:, 1:-2], n_q, table, pos, *odd, norm[1:], norm[1:], q_out=q2)
    assert torch.equal(q, q2) and torch.equal(kc, odd[0]) and torch.equal(vc, odd[1])


def test_rows_past_32_bit_offsets():
    """A cache of more than 2^32 elements: its last row."""
    d, L = 128, 1 << 20
    big = torch.empty(1, 1, 33 * L, d, dtype=torch.bfloat16, device="cuda")
    small = torch.zeros(1, 1, 33 * L, d, dtype=torch.bfloat16, device="cuda")[:, :, :, :d]
    assert big.numel() > 1 << 32
    qkv = _randn(_gen(5), 1, 3 * d, dtype=torch.bfloat16)
    pos = torch.tensor([33 * L - 1], dtype=torch.int32, device="cuda")
    table = ops.rope_table(pos, d, 1e6)
    ops.norm_rope_kv_append(qkv, 1, table, pos, big, small)
    k, v = big[0, 0, -1], small[0, 0, -1]
    assert torch.equal(v, qkv[0, 2 * d:])
    (_, _, kr, kt), _ = _reference(qkv, table, 1, 1, d, None, None, 0.0)
    _close(k, kr[0, 0], (kt + HALF[torch.bfloat16] * (kr.abs() + kt))[0, 0])


def test_captured_and_replayed():
    """In a graph on a stream of its own: replays follow the positions and tokens that its tensors hold."""
    g, B, n_q, n_k, n_v, d, L = _gen(6), 3, 4, 1, 2, 64, 32
    qkv, pos = _randn(g, B, 7 * d, dtype=torch.bfloat16), torch.zeros(B, dtype=torch.int32, device="cuda")
    table, one = torch.empty(B, d // 2, 2, device="cuda"), torch.ones(d, dtype=torch.bfloat16, device="cuda")
    kc, vc = (torch.zeros(B, h, L, d, dtype=torch.bfloat16, device="cuda") for h in (n_k, n_v))
    q = torch.empty(B, n_q, d, dtype=torch.bfloat16, device="cuda")

    def step():
        ops.rope_table(pos, d, 1e4, out=table)
        ops.norm_rope_kv_append(qkv, n_q, table, pos, kc, vc, one, one, q_out=q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        qkv.copy_(_randn(g, B, 7 * d, dtype=torch.bfloat16))
        pos.fill_(5 + i)
        graph.replay()
        got = q.clone(), kc.clone(), vc.clone()
        q.zero_()
        step()
        assert torch.equal(got[0], q) and torch.equal(got[1], kc) and torch.equal(got[2], vc)
        torch.cuda.synchronize()
    assert kc[:, :, 5:8].abs().sum(-1).min() > 0 and not kc[:, :, 8:].any()
