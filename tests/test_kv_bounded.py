"""Bounded decoders on the CPU: head groups that are refused when the decoder is built, not at its first step."""
from dataclasses import replace

import pytest

from saga_amd.decoder import DecoderShape, SagaDecoder

TINY = DecoderShape(2, 64, 4, 1, 2, 64, 128, 256, 1e4, 1e-6)


@pytest.mark.parametrize("n_q,n_k", [(18, 1), (34, 2), (40, 2)])
def test_wide_head_groups_of_16_bit_caches_are_refused(n_q, n_k):
    wide = replace(TINY, n_q=n_q, n_k=n_k)
    with pytest.raises(ValueError, match="16 query heads per key head"):
        SagaDecoder(wide, 1, 16, mode="dense", device="cpu", kv_budget=8)
    SagaDecoder(wide, 1, 16, mode="dense", device="cpu", kv_budget=8, kv_fp8_block=32)
    SagaDecoder(replace(wide, n_q=16 * n_k), 1, 16, mode="dense", device="cpu", kv_budget=8)
