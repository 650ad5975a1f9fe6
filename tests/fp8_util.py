"""The 8-bit cache of include/saga_amd.h in 64-bit arithmetic, position by position as written there, and random data."""
import math

import torch

F8 = torch.float8_e4m3fn


def grid(device="cpu"):
    """The 127 numbers from 0 to 448, by code."""
    return torch.arange(127, dtype=torch.uint8, device=device).view(F8).double()


def nearest(x):
    """Codes (uint8) of the e4m3 numbers nearest to x (|x| <= 448, or NaN), ties to the even code."""
    g, a = grid(x.device), x.double().abs().nan_to_num(0.0).contiguous()
    hi = torch.searchsorted(g, a).clamp(1, 126)
    under, over = a - g[hi - 1], g[hi] - a
    code = torch.where((over < under) | ((over == under) & (hi % 2 == 0)), hi, hi - 1)
    code = code + torch.where(torch.signbit(x), 128, 0)
    return torch.where(x.isnan(), 127, code).to(torch.uint8)


def opened(codes):
    return codes.view(F8).double()


def scale_of(top):
    """2^(floor(log2 top) - 5), at least 2^-100; 0 of 0."""
    if top == 0:
        return 0.0
    return math.ldexp(1.0, max(math.frexp(top)[1] - 6, -100))


def finite_top(x):
    a = x.double().abs()
    return float(torch.where(a.isfinite(), a, torch.zeros_like(a)).max())


def over(x, s):
    """x / s as it is rounded: NaN for what is not finite, 0 under the scale 0."""
    y = x.double() / s if s > 0 else x.double() * 0.0
    return torch.where(x.isfinite(), y, torch.full_like(y, float("nan")))


def append(codes, scales, block, start, x):
    """x [n, d] at positions start .. of one head's codes [L, d] and scales [blocks], in place."""
    n, at = x.shape[0], 0
    while at < n:
        p = start + at
        first = p // block * block
        m = min(first + block - p, n - at)
        new, old = x[at:at + m], float(scales[p // block])
        top = finite_top(new)
        s = old if p > first and top <= 448 * old else scale_of(top)
        if s != old and p > first:
            codes[first:p] = nearest(opened(codes[first:p]) * (old / s if s > 0 else 0.0))
        codes[p:p + m] = nearest(over(new, s))
        scales[p // block] = s
        at += m


def quantise(x, block):
    """Codes and scales of x [..., L, d], whole blocks at a time."""
    L, d = x.shape[-2:]
    nb = -(-L // block)
    g = torch.nn.functional.pad(x.double(), (0, 0, 0, nb * block - L)).unflatten(-2, (nb, block))
    top = g.abs().amax((-1, -2))
    e = torch.frexp(top)[1]
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(top).cpu(), (e.cpu() - 6).clamp(min=-100)).to(top), torch.zeros_like(top))
    c = nearest(g / torch.where(s > 0, s, torch.ones_like(s))[..., None, None])
    return c.flatten(-3, -2)[..., :L, :].contiguous(), s.float()


def values(codes, scales, block, dtype=torch.float64):
    s = scales.to(dtype).repeat_interleave(block, -1)[..., : codes.shape[-2], None]
    return codes.view(F8).to(dtype) * s


def random_cache(g, b, k_h, v_h, L, d, block, device="cuda"):
    """Quantised normal data: keys with offsets and a few long dims, blocks of different sizes."""
    from saga_amd import ops
    parts = []
    for kind, h in (("k", k_h), ("v", v_h)):
        x = torch.randn(b, h, L, d, generator=g, device=device)
        if kind == "k":
            x = x * (1 + 3 * (torch.rand(d, generator=g, device=device) < 0.1)) + torch.randn(d, generator=g, device=device)
        else:
            size = torch.exp2(torch.randint(-3, 3, (b, h, -(-L // block), 1), generator=g, device=device).float())
            x = x * size.repeat_interleave(block, 2)[:, :, :L]
        parts += quantise(x, block)
    return ops.KVFP8(*parts, block)


def cache_values(cache, dtype=torch.float64):
    return (values(cache.k_codes, cache.k_scales, cache.block, dtype),
            values(cache.v_codes, cache.v_scales, cache.block, dtype))


def clone(cache):
    return type(cache)(*(t.clone() for t in cache[:4]), cache.block)


def bits(t):
    """Codes or scales to compare bit by bit; the two bytes that are NaN (0x7f, 0xff) stand for the same."""
    return torch.where(t == 0xff, 0x7f, t) if t.dtype == torch.uint8 else t.contiguous().view(torch.int32)


def same(a, b):
    return all(torch.equal(bits(x), bits(y)) for x, y in zip(a[:4], b[:4]))


def kept_positions(w, n, keep, recent):
    """The kept positions of one row of weights (a list), place by place."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    H = keep - recent
    rank = lambda p: (0, 0.0, p) if math.isnan(w[p]) else (1, -w[p], p)
    heavy = sorted(range(n - recent), key=rank)[:H]
    stay = {p for p in heavy if p < H}
    movers = iter(sorted(p for p in heavy if p >= H))
    return [p if p in stay else next(movers) for p in range(H)] + list(range(n - recent, n))
