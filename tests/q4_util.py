"""The 4-bit formats of include/saga_amd.h, one code at a time as written there, and random data in them."""
import torch


def key_nibble(i, d):
    """Nibble of dim i in a key row: dim 32 j + 8 s + e is nibble 8 (s d / 32 + j) + e."""
    j, s, e = i // 32, i % 32 // 8, i % 8
    return 8 * (s * (d // 32) + j) + e


def value_nibble(i, d):
    """Nibble of dim i in a value row: dim 16 e + c is nibble c d / 16 + e."""
    return i % 16 * (d // 16) + i // 16


def weight_nibble(r, k):
    """Nibble of row r (of 16), column k (of 128) in a weight unit."""
    i, q, e = k // 32, k % 32 // 8, k % 8
    return (16 * q + r) * 32 + 8 * i + (0, 2, 4, 6, 1, 3, 5, 7).index(e)


def _bytes(codes, order):
    """codes [..., n] (uint8) placed in nibbles order[i] of [..., n / 2] bytes."""
    out = torch.zeros_like(codes)
    out[..., torch.tensor(order)] = codes
    return out[..., 0::2] | (out[..., 1::2] << 4)


def _codes(b, order):
    nib = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    return nib[..., torch.tensor(order, device=b.device)]


def pack_row(codes, kind):
    d = codes.shape[-1]
    return _bytes(codes.cpu(), [(key_nibble if kind == "k" else value_nibble)(i, d) for i in range(d)]).to(codes.device)


def open_row(b, kind):
    d = 2 * b.shape[-1]
    return _codes(b, [(key_nibble if kind == "k" else value_nibble)(i, d) for i in range(d)])


def open_weight(codes, K):
    """[N, K] codes of a packed weight's [N/16, units, 1024] bytes."""
    c = _codes(codes, [weight_nibble(r, k) for r in range(16) for k in range(128)])
    c = c.reshape(codes.shape[0], codes.shape[1], 16, 128).transpose(1, 2)
    return c.reshape(codes.shape[0] * 16, -1)[:, :K]


def values(codes, scales, dtype=torch.float64):
    """s * c + z; scales [..., 2 * groups]."""
    sz = scales.unflatten(-1, (-1, 2)).to(dtype)
    c = codes.to(dtype).unflatten(-1, (sz.shape[-2], -1))
    return (c * sz[..., :1] + sz[..., 1:]).flatten(-2)


def weight_values(w):
    N, K = w.shape
    sz = w.scales.double().transpose(1, 2).reshape(N, K // w.group, 2)
    return values(open_weight(w.codes, K), sz.flatten(-2))


def step_down(h):
    """The next f16 below h (finite), by its bits."""
    b = h.view(torch.int16)
    return torch.where(b > 0, b - 1, torch.where((b & 0x7fff) == 0, torch.full_like(b, -32767), b + 1)).view(torch.float16)


def quantise(x, group):
    """Codes and scales [..., 2 * groups] of x [..., n] by the rule of include/saga_amd.h, in x's own precision."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    bad = ~(g.abs().amax(-1, keepdim=True) <= 65504)
    z = lo.half()
    z = torch.where(z.to(x.dtype) > lo, step_down(z), z)
    q = (hi - z.to(x.dtype)) / torch.full_like(hi, 15)
    s = q.half()
    s = torch.where(s.to(x.dtype) < q, -step_down(-s), s)
    c = ((g - z.to(x.dtype)) / torch.where(s == 0, torch.ones_like(s), s).to(x.dtype)).round().clamp(0, 15)
    nan = torch.full_like(s, float("nan"))
    sz = torch.cat([torch.where(bad, nan, s), torch.where(bad, nan, z)], -1).flatten(-2)
    return torch.where(bad, torch.zeros_like(c), c).to(torch.uint8).flatten(-2), sz


def random_cache(g, b, k_h, v_h, L, d, group, device="cuda"):
    """A cache of quantised normal data (keys with offsets and a few long dims); the parts of ops.KVQ4."""
    from saga_amd import ops
    parts = []
    for kind, h in (("k", k_h), ("v", v_h)):
        x = torch.randn(b, h, L, d, generator=g, device=device)
        if kind == "k":
            x = x * (1 + 3 * (torch.rand(d, generator=g, device=device) < 0.1)) + torch.randn(d, generator=g, device=device)
        c, sz = quantise(x, group)
        parts += [pack_row(c, kind), sz]
    return ops.KVQ4(*parts)


def cache_values(cache, dtype=torch.float64):
    return (values(open_row(cache.k_codes, "k"), cache.k_scales, dtype),
            values(open_row(cache.v_codes, "v"), cache.v_scales, dtype))
