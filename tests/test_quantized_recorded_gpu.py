"""Recorded library calls of the cache in 4 bits, run again with other lengths and inputs on another stream."""

import gc

import pytest
import torch

from dcp_amd import _lib
from dcp_amd.flash_attn_interface import quantized_cache_attention, quantized_cache_workspace_bytes
from dcp_amd.ops import paged_cache_tables, quantized_cache_pages, quantized_cache_read, quantized_cache_write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 9]])
def test_a_recorded_step_is_run_again(gpu, new):
    size, batch, heads, kv_heads, d, n = 16, len(new), 8, 2, 64, sum(new)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cache = quantized_cache_pages(150, size, kv_heads, d, gpu)
    slots = torch.arange(150 * size, device=gpu)
    old = torch.randn(2, 150 * size, kv_heads, d, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(gpu)
    quantized_cache_write(old[0], old[1], slots, cache)
    pages = torch.randperm(150, generator=torch.Generator().manual_seed(n)).int().to(gpu)
    table, free = pages[: 20 * batch].view(batch, 20).clone(), pages[20 * batch : 20 * batch + 30].clone()
    lens, added = i32(100, 40, 0), i32(*new)
    q, k, v = (torch.empty(n, h, d, dtype=torch.bfloat16, device=gpu) for h in (heads, kv_heads, kv_heads))
    made = paged_cache_tables(lens, added, table.clone(), free, size, n)
    out, lse, back = torch.empty_like(q), torch.empty(heads, n, device=gpu), (torch.empty_like(k), torch.empty_like(v))
    own = dict(cu_seqlens_q=made.cu_seqlens, max_seqlen_q=max(new), max_seqlen_k=300)
    args = (q, cache, table, made.seq_lens)
    workspace = torch.empty(max(quantized_cache_workspace_bytes(*args, **own), 1), dtype=torch.uint8, device=gpu)

    def step():
        paged_cache_tables(lens, added, table, free, size, n, out=made)
        quantized_cache_write(k, v, made.slot_mapping, cache)
        quantized_cache_attention(*args, **own, out=out, lse=lse, workspace=workspace)
        quantized_cache_read(cache, made.slot_mapping, q.dtype, out=back)

    def fill(turn):
        lens.copy_(torch.tensor([[100, 40, 0], [3, 0, 17], [230, 200, 64]][turn % 3], dtype=torch.int32))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(turn)))

    state = (cache, table)
    start = [t.clone() for t in state]
    fill(0)
    recording, stream = _lib.Recording(), torch.cuda.Stream()
    assert recording.begin()
    try:
        step()
    finally:
        assert recording.end()
    assert recording.size() == 4
    gc.collect()  # (the calls' own arguments are not to be what their packed form pointed to)
    torch.cuda.synchronize()
    for turn in (0, 1, 2, 1):
        fill(turn)
        results = []
        for again in (False, True):
            for t, was in zip(state, start):
                t.copy_(was)
            for t in (out, lse, *back, *made):
                t.fill_(7)
            torch.cuda.synchronize()
            if again:
                recording.run(0, 4, stream.cuda_stream)
            else:
                step()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*state, out, lse, *back, *made)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), turn
        assert not torch.isnan(results[0][2]).any() and (results[0][2] != 7).any()
        assert (results[0][4] - k).abs().max() < k.abs().max() / 4  # (a code is off by less than a quarter of its block's largest)
