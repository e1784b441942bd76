"""What rounding the weights of attention over a cache in 4 bits may not do."""

import pytest
import torch

from dcp_amd.flash_attn_interface import quantized_cache_attention
from dcp_amd.ops import quantized_cache_pages, quantized_cache_write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beside", [3, 100])
@pytest.mark.parametrize("singles", [4, 70])
@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("longest", [64, 100000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_single_token_beside_a_prompt_is_rounded_as_alone(gpu, dtype, longest, group, singles, beside):
    """280 keys: 279 of weight 1 and value 0, and behind the first of them one of weight w from 2^12.5 to 2^13.5 and value 1: w / (w + 279).
    w is rounded by up to eps / 2 for the product.  Alone, a single token's sum has the rounded w as well, so that 279 / (w + 279) < 0.046 of that
    is left, beside half a step of the result (eps / 4 below 1) and sums in 32 bits.  The same holds where a request of more rows than the kernel of
    few rows takes is in the batch (3 tokens: tiles of 64 rows of 16 heads; 100: of 128), and where the host only says that there may be one."""
    kv_heads, d, n = 2, 64, 280
    k, v = (torch.zeros(n, kv_heads, d, dtype=dtype, device=gpu) for _ in range(2))
    k[270, :, 0], k[270, :, 1], v[270] = 6.0, 0.5, 1.0
    cache = quantized_cache_pages(18, 16, kv_heads, d, gpu)
    quantized_cache_write(k, v, torch.arange(n, device=gpu), cache)
    g = torch.Generator().manual_seed(1)
    q = torch.zeros(singles + beside, kv_heads * group, d)
    q[..., 0], q[..., 1] = 11.5625, torch.rand(q.shape[:2], generator=g) * 10
    q = q.to(dtype)
    w = torch.exp((6 * q[:singles, :, 0].double() + 0.5 * q[:singles, :, 1].double()) * d**-0.5)
    assert w.log2().min() > 12.5 and w.log2().max() < 13.5
    eps = torch.finfo(dtype).eps
    for batch in (singles, singles + 1):
        lens = torch.full((batch,), n, dtype=torch.int32, device=gpu)
        table = torch.arange(18, dtype=torch.int32, device=gpu).expand(batch, 18).contiguous()
        cu = torch.tensor([*range(singles + 1), singles + beside][: batch + 1], dtype=torch.int32, device=gpu)
        tokens = int(cu[-1])
        out, lse = quantized_cache_attention(q[:tokens].to(gpu), cache, table, lens, cu_seqlens_q=cu, max_seqlen_q=beside, max_seqlen_k=longest)
        off = (out[:singles].double().cpu() - (w / (w + n - 1))[..., None]).abs().max()
        assert off <= eps / 4 + 0.046 * eps / 2 + 2.0**-16, (batch, float(off / eps))
        assert (lse[:, :singles].double().cpu().T - (w + n - 1).log()).abs().max() <= 2.0**-18
