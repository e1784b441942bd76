"""Attention over a cache in 4 bits whose pages are longer than 2^31 bytes."""

import pytest
import torch

from dcp_amd.flash_attn_interface import quantized_cache_attention
from dcp_amd.ops import quantized_cache_write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [None, 64])
@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_31_bits_in_a_page(gpu, window, new):
    """One page of 15.84 million tokens: its last ones begin 2.15 GB behind its start.  All keys are 0, so every visible one has weight 1, and
    of the values all are 0 but the last 16, which are 2^20: the sum of so many ones is exact in 32 bits, the result rounded to bf16 (half a step,
    2^-8), the quotient and the joining of pieces off by less than 2^-14."""
    blocks, d = 990_000, 128
    n = blocks * 16
    assert blocks * 17 * d > 2**31 and n < 2**24
    cache = torch.zeros(1, 1, blocks, 17 * d, dtype=torch.uint8, device=gpu)
    v = torch.full((16, 1, d), 2.0**20, dtype=torch.bfloat16, device=gpu)
    quantized_cache_write(torch.zeros_like(v), v, torch.arange(n - 16, n, device=gpu), cache)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    q = torch.randn(new, 2, d, device=gpu).to(torch.bfloat16)
    out, lse = quantized_cache_attention(q, cache, i32(0)[None], i32(n), cu_seqlens_q=i32(0, new), max_seqlen_q=new, window=window)
    at = torch.arange(n - new, n, dtype=torch.float64)  # of the tokens
    seen = at + 1 if window is None else torch.full_like(at, window)
    truth = 2.0**20 * (at - (n - 17)).clamp(min=0) / seen
    assert ((out.double().cpu() - truth[:, None, None]).abs() <= (2.0**-8 + 2.0**-14) * truth[:, None, None]).all()
    assert ((lse.double().cpu() - seen.log()).abs() <= 2.0**-20 * (1 + seen.log())).all()
