"""What SagaDecoder appends, on the GPU: every layer's keys and values of a prompt and of steps, before and after
evictions, against a 64-bit forward pass that computes them itself; the same pass with a mistake in it is told apart."""
import math

import pytest
import torch

from test_gpu_kv_decoder import _decoder, _held, _norm, _values

pytestmark = pytest.mark.gpu

MISTAKES = ("other layer's k_norm", "q_norm on keys", "no k_norm", "value heads swapped", "rotated by place", "keys not rotated")


def _forward64(m, ids, pos0, place0, caches, mistake=None, eps=None):
    """Per layer the keys [T, n_k, d] and values [T, n_v, d] of the tokens ids at positions pos0 .., which attend over the
    places up to place0 + their index of the caches, in 64 bits."""
    s, d, T = m.shape, m.shape.head_dim, len(ids)
    x = m.embed[ids].double()

    def turned(t, first):
        pos = torch.arange(first, first + T, device="cuda", dtype=torch.float64)
        ang = pos[:, None] * s.rope_theta ** (-2 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
        z = torch.complex(t[..., : d // 2], t[..., d // 2:]) * torch.polar(torch.ones_like(ang), ang)[:, None]
        return torch.cat([z.real, z.imag], -1)

    found = []
    for l in range(s.layers):
        qkv = (_norm(x, s.eps) * m.ln1[l].double() @ m.w_qkv[l].double().t() + m.b_qkv[l].double()).view(T, -1, d)
        q, k, v = qkv.split([s.n_q, s.n_k, s.n_v], 1)
        if s.qk_norm:
            q = _norm(q, s.eps) * m.q_norm[l].double()
            weight = {"other layer's k_norm": m.k_norm[(l + 1) % s.layers], "q_norm on keys": m.q_norm[l]}.get(mistake, m.k_norm[l])
            if mistake != "no k_norm":
                k = _norm(k, s.eps if eps is None else eps) * weight.double()
        if mistake == "value heads swapped":
            v = v.flip(1)
        if mistake != "keys not rotated":
            k = turned(k, place0 if mistake == "rotated by place" else pos0)
        q = turned(q, pos0)
        found.append((k, v))
        kc, vc = caches[l]
        o = torch.empty(T, s.n_q, d, dtype=torch.float64, device="cuda")
        for h in range(s.n_q):
            a = q[:, h] @ kc[h * s.n_k // s.n_q].t() / math.sqrt(d)
            last = place0 + torch.arange(T, device="cuda")
            a = a.masked_fill(torch.arange(kc.shape[1], device="cuda")[None] > last[:, None], -math.inf)
            o[:, h] = torch.softmax(a, -1) @ vc[h * s.n_v // s.n_q]
        x = x + o.view(T, -1) @ m.w_o[l].double().t()
        gu = _norm(x, s.eps) * m.ln2[l].double() @ m.w_gu[l].double().t()
        g, u = gu.split(s.intermediate, -1)
        x = x + (g * torch.sigmoid(g) * u) @ m.w_d[l].double().t()
    return found


def _off(m, ref, place0, row, step):
    """How far, of their bounds, what row `row` holds from place0 on is from ref: the largest over layers, kinds and
    tokens.  `step`: half a step of the decoder's type and how many of them a layer adds.  A layer's residual
    stream is off by `step` a layer below it, its own norm, projection and store by 4 more; a norm of keys doubles
    what reaches it.  8 bits: one rounding, 2^-4 of a value and 2^-10 of its scale at most."""
    worst = 0.0
    for l, (kinds, held) in enumerate(zip(ref, _values(m))):
        for i, (x, cache) in enumerate(zip(kinds, held)):
            T = x.shape[0]
            got = cache[row, :, place0:place0 + T].transpose(0, 1)
            size = x.norm(dim=-1)
            bound = size * 2 * (step[1] * l + 4) * step[0]
            if m.kv_fp8_block:
                c = m.kv.layer(l)
                scales = (c.v_scales if i else c.k_scales)[row].double()
                block = (place0 + torch.arange(T, device="cuda")) // m.kv_fp8_block
                bound = bound + 2.0 ** -4 * (size + bound) + 2.0 ** -10 * math.sqrt(x.shape[-1]) * scales[:, block].t()
            worst = max(worst, float(((got - x).norm(dim=-1) / bound).max()))
    return worst


def _check(m, ids, pos0, place0, row, step):
    """The rows of the tokens ids; those of a pass with a mistake, where it makes a difference, are none of them."""
    held = _held(m, row, place0 + len(ids))
    assert _off(m, _forward64(m, ids, pos0, place0, held), place0, row, step) <= 1
    for mistake in MISTAKES:
        if not m.shape.qk_norm and "norm" in mistake or pos0 == place0 and mistake == "rotated by place":
            continue
        if mistake == "keys not rotated" and pos0 == 0 and len(ids) == 1:
            continue
        assert _off(m, _forward64(m, ids, pos0, place0, held, mistake), place0, row, step) > 1, mistake


@pytest.mark.parametrize("shape", ["qwen", "llama", "groups"])
@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("block", [0, 32, 64])
def test_rows_of_a_prompt_and_of_steps(shape, qk_norm, block):
    m = _decoder(shape, 2, 96, qk_norm, kv_fp8_block=block)
    ids = torch.randint(0, m.shape.vocab, (37,), generator=torch.Generator().manual_seed(1)).cuda()
    m.prefill(ids)
    _check(m, ids, 0, 0, 0, (2.0 ** -8, 10))
    for i in range(3):
        token = m.tokens.clone()
        m.step(calibrate=False)
        _check(m, token[1:], 37 + i, 37 + i, 1, (2.0 ** -8, 10))


@pytest.mark.parametrize("shape,qk_norm,block", [("qwen", True, 0), ("groups", True, 32), ("llama", False, 64), ("qwen", True, 128)])
@pytest.mark.parametrize("graphs", [False, True])
def test_rows_of_steps_behind_evictions(shape, qk_norm, block, graphs):
    """A token's place is no longer its position: it is rotated by the latter."""
    m = _decoder(shape, 2, 61, qk_norm, kv_fp8_block=block, kv_budget=33, kv_recent=8)
    m.prefill(torch.randint(0, m.shape.vocab, (45,), generator=torch.Generator().manual_seed(2)))
    if graphs:
        m.capture()
    for i in range(50):
        token = m.tokens.clone()
        if graphs:
            m.replay(i)
        else:
            m.step(calibrate=False)
        if i in (0, 15, 16, 30, 49):
            place = int(m.slot[0]) - 1
            assert (place == 45 + i) == (i < 16)
            _check(m, token[1:], 45 + i, place, 1, (2.0 ** -8, 10))


def test_rows_of_a_float32_decoder_whose_heads_are_small():
    """f32, heads as small as sqrt(eps), so that a norm's eps counts: products of up to 640 terms, sums off by at most 640
    steps of 2^-24 each, 5 of them a layer."""
    m = _decoder("groups", 2, 64, True, dtype=torch.float32)
    for w in m.w_qkv:
        w.mul_(2.0 ** -7)
    ids = torch.randint(0, m.shape.vocab, (20,), generator=torch.Generator().manual_seed(4)).cuda()
    step = (640 * 2.0 ** -24, 5)
    m.prefill(ids)
    _check(m, ids, 0, 0, 0, step)
    token = m.tokens.clone()
    m.step(calibrate=False)
    _check(m, token[:1], 20, 20, 0, step)
    held = _held(m, 0, 21)
    for eps in (0.0, 1e-6, 2e-5):  # (the shape's is 1e-5)
        assert _off(m, _forward64(m, token[:1], 20, 20, held, eps=eps), 20, 0, step) > 1
