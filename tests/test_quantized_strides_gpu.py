"""Keys and values at strides of their own, written into a cache in 4 bits and read out of it on the GPU."""

import pytest
import torch

from dcp_amd import _lib
from dcp_amd.ops import quantized_cache_pages, quantized_cache_read, quantized_cache_write

pytestmark = pytest.mark.gpu

LAYOUTS = {  # of [n, heads, d] in wider memory filled with `fill`
    "dense": lambda n, h, d, new: new(n, h, d),
    "fused": lambda n, h, d, new: new(n, 3 * h + 2, d)[:, h + 1 : 2 * h + 1],
    "by_head": lambda n, h, d, new: new(h, n, d).transpose(0, 1),
    "padded": lambda n, h, d, new: new(n, h, d + 8)[..., :d],
    "one_token_apart": lambda n, h, d, new: new(h, 2 * n + 1, d)[:, 1::2].transpose(0, 1),
}
PAIRS = [("dense", "fused"), ("fused", "by_head"), ("by_head", "dense"), ("padded", "one_token_apart")]


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("n,heads", [(1, 4), (1, 1), (37, 1), (70, 5)])
@pytest.mark.parametrize("of_k,of_v", PAIRS)
def test_strides_that_differ(gpu, dtype, d, n, heads, of_k, of_v):
    """Byte for byte as from dense copies, and nothing beside the rows is written."""
    new = lambda *shape: torch.full(shape, 7.0, dtype=dtype, device=gpu)
    k, v = (LAYOUTS[of](n, heads, d, new) for of in (of_k, of_v))
    k.copy_(torch.randn(k.shape, generator=torch.Generator().manual_seed(n)))
    v.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(n + 1)))
    slots = torch.randperm(96, generator=torch.Generator().manual_seed(n))[:n].to(gpu)
    want, cache = (quantized_cache_pages(3, 32, heads, d, gpu) for _ in range(2))
    quantized_cache_write(k.contiguous(), v.contiguous(), slots, want)
    quantized_cache_write(k, v, slots, cache)
    assert torch.equal(cache, want) and (cache != 0).any()
    stores = []
    kept = lambda *shape: stores.append(new(*shape)) or stores[-1]
    out = LAYOUTS[of_v](n, heads, d, kept), LAYOUTS[of_k](n, heads, d, kept)
    got = quantized_cache_read(cache, slots, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for x, y, store in zip(out, quantized_cache_read(cache, slots, dtype), stores):
        assert torch.equal(x, y)
        x.fill_(7)
        assert (store == 7).all()


def test_an_odd_stride_of_one_token(gpu):
    k, v = (torch.randn(1000, dtype=torch.bfloat16, device=gpu).as_strided((1, 2, 64), (token, 64, 1)) for token in (3, 997))
    want, cache, slots = quantized_cache_pages(1, 16, 2, 64, gpu), quantized_cache_pages(1, 16, 2, 64, gpu), torch.tensor([5], device=gpu)
    quantized_cache_write(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format), slots, want)
    quantized_cache_write(k, v, slots, cache)
    assert torch.equal(cache, want) and (cache != 0).any()


def test_recorded(gpu):
    """A recording of calls whose strides differ is one call each, run again over what is there by then."""
    k, fused = torch.empty(9, 2, 64, dtype=torch.bfloat16, device=gpu), torch.empty(9, 8, 64, dtype=torch.bfloat16, device=gpu)
    v, cache, slots = fused[:, 3:5], quantized_cache_pages(2, 16, 2, 64, gpu), torch.arange(3, 12, device=gpu)
    out = torch.empty_like(fused)[:, 1:3], torch.empty_like(k)
    recording = _lib.Recording()
    assert recording.begin()
    try:
        quantized_cache_write(k, v, slots, cache)
        quantized_cache_read(cache, slots, out=out)
    finally:
        assert recording.end()
    assert recording.size() == 2
    for turn in range(3):
        k.copy_(torch.randn(k.shape, generator=torch.Generator().manual_seed(turn)))
        fused.copy_(torch.randn(fused.shape, generator=torch.Generator().manual_seed(turn + 10)))
        recording.run(0, 2, torch.cuda.current_stream().cuda_stream)
        want = quantized_cache_pages(2, 16, 2, 64, gpu)
        quantized_cache_write(k.contiguous(), v.contiguous(), slots, want)
        assert torch.equal(cache, want) and all(torch.equal(a, b) for a, b in zip(out, quantized_cache_read(want, slots)))
