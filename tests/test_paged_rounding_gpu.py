"""What rounding the weights of paged attention may not do."""

import pytest
import torch

from dcp_amd.flash_attn_interface import shared_prefix_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("longest_q", [1, 40, None])
@pytest.mark.parametrize("shared", [True, False])
def test_a_prefix_of_equal_values_is_returned_as_it_is(gpu, dtype, head_dim, longest_q, shared):
    """O of a prefix is divided by the sum of the weights that went into it, the rounded ones, whichever launch takes it: values that
    are all the same come back unchanged.  (Sums of at most 300 terms in 32 bits, their quotients and the joining of at most 64
    shares: off by less than 600 * 2^-23 < 2^-13 relative, where half a step of the result is 2^-9 of it or more in bf16 and 2^-12 in fp16.)
    There are two different keys, one in thirty and the rest, so that in every share the errors of the rest's weights are the same and do
    not cancel."""
    heads, kv_heads, size, n_keys, new = 8, 2, 16, 300, 40
    g = torch.Generator().manual_seed(head_dim)
    n_pages = -(-n_keys // size)
    k = torch.randn(2, kv_heads, head_dim, generator=g)[(torch.arange(n_pages * size) % 30 > 0).long()]
    value = (1 + torch.rand(kv_heads, head_dim, generator=g)).to(dtype)
    cache = torch.stack([k.to(dtype), value.expand(n_pages * size, -1, -1)], 1).view(n_pages, size, 2, kv_heads, head_dim).to(gpu)
    tokens = 2 * new if shared else new
    q = torch.randn(tokens, heads, head_dim, generator=g).to(dtype).to(gpu)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    requests = tokens // new
    out, _ = shared_prefix_attention(q, cache[:, :, 0], cache[:, :, 1], torch.arange(n_pages, dtype=torch.int32, device=gpu)[None], i32(n_keys),
                                     i32(0, requests), torch.full((requests, 1), -1, dtype=torch.int32, device=gpu), i32(*[0] * requests),
                                     cu_seqlens_q=i32(*range(0, tokens + 1, new)), max_seqlen_q=longest_q, max_seqlen_k=16, max_prefix_len=n_keys)
    want = value.to(gpu).repeat_interleave(heads // kv_heads, 0).expand(tokens, -1, -1)
    assert torch.equal(out, want), f"{int((out != want).sum())} of {out.numel()} changed"
