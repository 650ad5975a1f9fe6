"""KV-cache layout, allocation and capacity planning for SAGA decoders.

The reference keeps separate per-layer key and value caches, K [B, k_h, Lmax,
d] and V [B, v_h, Lmax, d] (speedup.py:119-139, the StaticCache layout of
transformers cache_utils.py:455-487), with k_h < v_h in SAGA models.  This
build keeps the same per-layer layout and stores all layers in one tensor per
kind: K [layers, B, k_h, Lmax, d] and V [layers, B, v_h, Lmax, d].
  * contiguous, so each layer's cache is a view in the reference layout (the
    kernels take it in place; a d = 128 bf16 row is 256 bytes);
  * each tensor starts 256-byte aligned (caching allocator blocks are);
  * one allocation per kind: the 28 layers of a 1.5B-shaped model at batch
    8 and 32k context are two tensors of 1.9 and 3.8 GB.

With bits=4 a cache holds 4-bit codes with an f16 scale and offset per group
of 32 or 64 dims (ops.KVQ4 per layer): 4.5 or 5 bits a value, so 3.2 to 3.6
times the positions.  With fp8_block it holds e4m3 numbers with a scale per
head and block of that many positions (ops.KVFP8 per layer): twice the positions.

plan_capacity() answers how long a context, or how large a batch, fits on one
GPU next to the decode weights and workspaces: an MI355X has 288 GB of HBM3E.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

HBM_BYTES_MI355X = 288 * 10**9
MAX_GROUP = 16  # query heads per key head that ops.attention_weights takes, as all attention over 16-bit caches


def _es(dtype) -> int:
    return torch.tensor([], dtype=dtype).element_size()


def _check_bits(name: str, bits: int) -> None:
    if bits not in (4, 16):
        raise ValueError(f"{name} must be 16 or 4, got {bits}")


def _check_q4_rows(d: int, group: int) -> None:
    if d not in (64, 128) or group not in (32, 64):
        raise ValueError(f"a 4-bit cache needs a head dim of 64 or 128 and groups of 32 or 64, got {d} and {group}")


def check_fp8_decoder(shape, dtype, kv_fp8_block: int, kv_bits: int = 16) -> None:
    """ValueError for 8-bit caches, or norms of queries and keys, that SagaDecoder does not take."""
    if kv_fp8_block:
        _check_fp8_rows(shape.head_dim, kv_fp8_block)
        if kv_bits != 16:
            raise ValueError("kv_fp8_block and kv_bits=4 exclude each other")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("kv_fp8_block needs bf16 or f16")
    if shape.qk_norm and (shape.head_dim not in (64, 128) or kv_bits != 16):
        raise ValueError("norms of queries and keys need a head dim of 64 or 128 and 16- or 8-bit caches")


def check_bounded_decoder(shape, max_len: int, kv_bits: int, kv_fp8_block: int, kv_budget: int, kv_recent: int) -> None:
    """ValueError for a bounded cache that SagaDecoder does not take."""
    if kv_budget and (kv_bits != 16 or shape.head_dim not in (64, 128)):
        raise ValueError("kv_budget needs 16- or 8-bit caches and a head dim of 64 or 128")
    if kv_budget and not kv_fp8_block and shape.n_q > MAX_GROUP * shape.n_k:
        raise ValueError(f"kv_budget over 16-bit caches takes at most {MAX_GROUP} query heads per key head")
    if (kv_budget or kv_recent) and not (0 < kv_budget < max_len and 0 <= kv_recent <= kv_budget):
        raise ValueError("kv_budget must lie between 1 and max_len - 1, kv_recent between 0 and kv_budget")


def _check_fp8_rows(d: int, block: int) -> None:
    if d not in (64, 128) or block not in (32, 64, 128):
        raise ValueError(f"an 8-bit cache needs a head dim of 64 or 128 and blocks of 32, 64 or 128 positions, got {d} and {block}")


def projection_shapes(shape):
    """(rows, columns) of a layer's q/k/v, o, gate/up and down projections, and of the LM head."""
    s = shape
    return ((s.qkv_width, s.hidden), (s.hidden, s.n_q * s.head_dim), (2 * s.intermediate, s.hidden),
            (s.hidden, s.intermediate), (s.vocab, s.hidden))


def skinny_gemm_supported(shape, batch: int, dtype) -> bool:
    """Whether a decoder's projections run through the skinny GEMM (ops.gemv, ops.gemv_q4)."""
    return (batch <= 32 and dtype == torch.bfloat16 and shape.hidden % 32 == 0 and shape.intermediate % 32 == 0
            and (shape.n_q * shape.head_dim) % 32 == 0 and shape.qkv_width % 16 == 0 and shape.vocab % 16 == 0)


def check_q4_decoder(shape, batch: int, dtype, kv_bits: int, kv_group: int, weight_bits: int, weight_group: int) -> None:
    """ValueError for caches or weights in 4 bits that SagaDecoder does not take."""
    _check_bits("kv_bits", kv_bits)
    _check_bits("weight_bits", weight_bits)
    if kv_bits == 4:
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("kv_bits=4 needs bf16 or f16")
        _check_q4_rows(shape.head_dim, kv_group)
    if weight_bits == 4:
        if weight_group not in (32, 64, 128):
            raise ValueError(f"weight_group: 4-bit weights need groups of 32, 64 or 128 columns, got {weight_group}")
        if not skinny_gemm_supported(shape, batch, dtype) or any(k % weight_group for _, k in projection_shapes(shape)):
            raise ValueError("weight_bits=4 needs bf16, a batch of at most 32 and widths that are multiples of weight_group")


def kv_cache_bytes(shape, batch: int, max_len: int, dtype=torch.bfloat16, bits: int = 16, group: int = 64,
                   fp8_block: int = 0) -> int:
    """Bytes of the K and V caches of every layer; bits 4: codes and the scales of groups of `group` dims; fp8_block:
    e4m3 numbers and the scales of blocks of so many positions."""
    _check_bits("bits", bits)
    d = shape.head_dim
    if bits == 4:
        _check_q4_rows(d, group)
    if fp8_block:
        _check_fp8_rows(d, fp8_block)
        return shape.layers * batch * (shape.n_k + shape.n_v) * (max_len * d + -(-max_len // fp8_block) * 4)
    row = d * _es(dtype) if bits == 16 else d // 2 + 4 * (d // group)
    return shape.layers * batch * (shape.n_k + shape.n_v) * max_len * row


def decode_weight_bytes(shape, dtype=torch.bfloat16, decode_copies: bool = True, bits: int = 16,
                        group: int = 64) -> int:
    """Weights of a decoder of this shape: embedding (tied LM head), per-layer
    q/k/v (+ bias), o, gate/up and down projections, norms.  decode_copies:
    plus the decode-layout copies the skinny GEMM reads (norm-folded q/k/v and
    gate/up, packed o and down, normed LM head), with bits=4 in codes and
    scales (rows padded to 128 columns).  A decoder releases the row-major
    projections once its copies are made: both are there until then."""
    _check_bits("bits", bits)
    if bits == 4 and (group not in (32, 64, 128) or any(k % group for _, k in projection_shapes(shape))):
        raise ValueError(f"4-bit weights need groups of 32, 64 or 128 columns that divide every width, got {group}")
    es = _es(dtype)
    s = shape
    per_layer = (s.qkv_width * s.hidden + s.qkv_width + s.hidden * s.n_q * s.head_dim + 2 * s.intermediate * s.hidden
                 + s.hidden * s.intermediate + 2 * s.hidden + (2 * s.head_dim if s.qk_norm else 0))
    base = (s.vocab * s.hidden + s.layers * per_layer + s.hidden) * es
    if not decode_copies:
        return base

    def copy(n, k):
        return n * k * es if bits == 16 else n * ((k + 127) // 128 * 64 + 4 * (k // group))

    *layer, head = (copy(n, k) for n, k in projection_shapes(s))
    return base + s.layers * sum(layer) + head


def decode_workspace_bytes(shape, batch: int, max_len: int, top_n: int, kv_bits: int = 16,
                           weight_bits: int = 16, kv_fp8_block: int = 0, kv_budget: int = 0, kv_recent: int = 0,
                           dtype=torch.bfloat16) -> int:
    """Atop-N and dense decode workspaces of one layer call (shared by all
    layers; a 4- or 8-bit cache: its dense workspace), the projections' (of 16-
    or 4-bit weights), plus the per-step activations and the threshold table;
    of a bounded cache besides the weights that its positions (and a prompt's)
    gathered, the workspaces that gather them, and the eviction's."""
    from . import _lib
    lib = _lib.load()
    s = shape
    if kv_bits == 4:
        ws = lib.saga_dense_q4_workspace_bytes(batch, s.n_q, max_len, s.head_dim)
    elif kv_fp8_block:
        ws = lib.saga_dense_fp8_workspace_bytes(batch, s.n_q, max_len, s.head_dim, 1 if kv_budget else 0)
    else:
        ws = lib.saga_atopn_workspace_bytes(batch, s.n_q, s.n_k, max_len, s.head_dim, min(2 * top_n, max_len))
        ws += lib.saga_dense_workspace_bytes(batch, s.n_q, max_len, s.head_dim)
    if weight_bits == 4:
        ws += max(lib.saga_gemv_q4_workspace_bytes(batch, n, k) for n, k in projection_shapes(s))
    else:
        ws += lib.saga_gemv_workspace_bytes(batch, s.hidden, s.intermediate)
    if kv_budget:
        G, row = math.gcd(s.n_k, s.n_v), s.head_dim * (1 if kv_fp8_block else _es(dtype))
        ws += 2 * s.layers * batch * G * max_len * 4
        ws += lib.saga_evict_workspace_bytes(batch, G, kv_budget, kv_recent, s.n_k + s.n_v, row, 1)
        if not kv_fp8_block:
            ws += lib.saga_attention_weights_workspace_bytes(batch, s.n_q, s.n_k, max_len)
    ws += s.layers * batch * s.n_q * 4
    ws += batch * (3 * s.hidden + s.qkv_width + 2 * s.intermediate + s.vocab) * 2
    return int(ws)


@dataclass(frozen=True)
class CapacityPlan:
    batch: int
    max_len: int
    kv_bytes: int
    weight_bytes: int
    workspace_bytes: int
    budget_bytes: int

    @property
    def total_bytes(self) -> int:
        return self.kv_bytes + self.weight_bytes + self.workspace_bytes

    def __str__(self) -> str:
        g = 1e9
        return (f"batch {self.batch} x {self.max_len} positions: KV {self.kv_bytes / g:.1f} GB + weights "
                f"{self.weight_bytes / g:.1f} GB + workspaces {self.workspace_bytes / g:.2f} GB = "
                f"{self.total_bytes / g:.1f} of {self.budget_bytes / g:.0f} GB")


def plan_capacity(shape, batch: Optional[int] = None, max_len: Optional[int] = None, budget_bytes: Optional[int] = None,
                  reserve_fraction: float = 0.05, top_n: int = 512, dtype=torch.bfloat16,
                  align: int = 256, kv_bits: int = 16, weight_bits: int = 16, group: int = 64,
                  kv_group: Optional[int] = None, weight_group: Optional[int] = None,
                  kv_fp8_block: int = 0, kv_budget: int = 0, kv_recent: int = 0) -> CapacityPlan:
    """The largest max_len for a given batch, or the largest batch for a given
    max_len (give exactly one), that fits budget_bytes (default: the current
    device's total memory, else 288 GB) minus reserve_fraction, next to the
    decode weights (with their decode copies) and workspaces.  max_len is
    rounded down to a multiple of `align` positions.  kv_bits, weight_bits:
    caches and decode copies in 4 bits, in groups of kv_group and weight_group
    (`group` where not given); kv_fp8_block: caches in 8 bits, in blocks of so
    many positions; kv_budget, kv_recent: a bounded cache of max_len places;
    what SagaDecoder refuses is refused, and a batch searched for ends at the
    32 rows that 4-bit weights take."""
    if (batch is None) == (max_len is None):
        raise ValueError("give exactly one of batch and max_len")
    kv_group, weight_group = kv_group or group, weight_group or group
    check_q4_decoder(shape, batch or 1, dtype, kv_bits, kv_group, weight_bits, weight_group)
    check_fp8_decoder(shape, dtype, kv_fp8_block, kv_bits)
    check_bounded_decoder(shape, 1 << 30 if max_len is None else max_len, kv_bits, kv_fp8_block, kv_budget, kv_recent)
    if budget_bytes is None:
        budget_bytes = (torch.cuda.get_device_properties(0).total_memory if torch.cuda.is_available()
                        else HBM_BYTES_MI355X)
    avail = int(budget_bytes * (1 - reserve_fraction))
    wbytes = decode_weight_bytes(shape, dtype, bits=weight_bits, group=weight_group)

    def fits(b: int, L: int) -> Optional[CapacityPlan]:
        if weight_bits == 4 and b > 32:
            return None
        kv = kv_cache_bytes(shape, b, L, dtype, kv_bits, kv_group, kv_fp8_block)
        ws = decode_workspace_bytes(shape, b, L, top_n, kv_bits, weight_bits, kv_fp8_block, kv_budget, kv_recent, dtype)
        if kv + wbytes + ws > avail:
            return None
        return CapacityPlan(b, L, kv, wbytes, ws, budget_bytes)

    best = None
    if batch is not None:
        lo, hi = 0, 1
        while fits(batch, hi * align) is not None and hi < (1 << 24):
            lo, hi = hi, hi * 2
        while hi - lo > 1:  # largest multiple of align that fits
            mid = (lo + hi) // 2
            if fits(batch, mid * align) is not None:
                lo = mid
            else:
                hi = mid
        best = fits(batch, lo * align) if lo > 0 else None
        if best is not None and kv_budget >= best.max_len:
            raise MemoryError(f"no cache of more than kv_budget {kv_budget} positions fits (at most {best.max_len})")
    else:
        lo, hi = 0, 1
        while fits(hi, max_len) is not None and hi < (1 << 20):
            lo, hi = hi, hi * 2
        while hi - lo > 1:
            mid = (lo + hi) // 2
            if fits(mid, max_len) is not None:
                lo = mid
            else:
                hi = mid
        best = fits(lo, max_len) if lo > 0 else None
    if best is None:
        raise MemoryError(f"nothing fits: weights alone are {wbytes / 1e9:.1f} GB of {avail / 1e9:.0f} GB")
    return best


class KVCache:
    """K [layers, B, k_h, Lmax, d] and V [layers, B, v_h, Lmax, d], zero-filled;
    layer(l) returns the reference-layout views (k [B, k_h, Lmax, d],
    v [B, v_h, Lmax, d]).  bits=4: 4-bit codes and scales (zeros) of groups of
    `group` dims; layer(l) returns ops.KVQ4 and k, v are None.  fp8_block: e4m3
    numbers and scales (zeros) of blocks of so many positions; layer(l) returns
    ops.KVFP8 and k, v are None."""

    def __init__(self, shape, batch: int, max_len: int, device="cuda", dtype=torch.bfloat16,
                 check_free: bool = True, bits: int = 16, group: int = 64, fp8_block: int = 0):
        dev = torch.device(device)
        d = shape.head_dim
        _check_bits("bits", bits)
        if fp8_block and bits != 16:
            raise ValueError("fp8_block and bits=4 exclude each other")
        need = kv_cache_bytes(shape, batch, max_len, dtype, bits, group, fp8_block)
        if check_free and dev.type == "cuda":
            free, _ = torch.cuda.mem_get_info(dev)
            if need > 0.8 * free:
                raise MemoryError(f"KV cache of {need / 2**30:.1f} GiB does not fit in {free / 2**30:.1f} GiB free "
                                  f"HBM (plan_capacity() gives the largest batch / context)")
        self.k = self.v = self.q4 = self.fp8 = None
        if fp8_block:
            from .ops import KVFP8
            blocks = -(-max_len // fp8_block)
            parts = [torch.zeros(shape.layers, batch, h, *row, device=dev, dtype=dt) for h in (shape.n_k, shape.n_v)
                     for row, dt in (((max_len, d), torch.uint8), ((blocks,), torch.float32))]
            self.fp8 = KVFP8(*parts, fp8_block)
        elif bits == 4:
            from .ops import KVQ4

            def zeros(heads, row, dt):
                return torch.zeros(shape.layers, batch, heads, max_len, row, device=dev, dtype=dt)

            self.q4 = KVQ4(*(zeros(h, row, dt) for h in (shape.n_k, shape.n_v)
                             for row, dt in ((d // 2, torch.uint8), (2 * d // group, torch.float16))))
        else:
            self.k = torch.zeros(shape.layers, batch, shape.n_k, max_len, d, device=dev, dtype=dtype)
            self.v = torch.zeros(shape.layers, batch, shape.n_v, max_len, d, device=dev, dtype=dtype)
        self.batch, self.max_len, self.bits = batch, max_len, bits

    @property
    def tensors(self):
        if self.fp8 is not None:
            return self.fp8[:4]
        return self.q4 if self.bits == 4 else (self.k, self.v)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tensors)

    def layer(self, l: int):
        if self.fp8 is not None:
            return type(self.fp8)(*(t[l] for t in self.fp8[:4]), self.fp8.block)
        return type(self.q4)(*(t[l] for t in self.q4)) if self.bits == 4 else (self.k[l], self.v[l])
