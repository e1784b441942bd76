"""Recorded library calls of the paged cache's operators, run again with other lengths and inputs on another stream."""

import gc

import pytest
import torch

from dcp_amd import _lib
from dcp_amd.flash_attn_interface import (paged_cache_attention, paged_cache_workspace_bytes, shared_prefix_attention,
                                          shared_prefix_workspace_bytes)
from dcp_amd.ops import paged_cache_tables, paged_cache_write

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 9]])
def test_a_recorded_step_is_run_again(gpu, new):
    size, batch, heads, kv_heads, d, n = 16, len(new), 8, 2, 64, sum(new)
    g = torch.Generator(device=gpu).manual_seed(n)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cache = torch.randn(150, size, 2, kv_heads, d, device=gpu, generator=g).to(torch.bfloat16)
    k_cache, v_cache = cache[:, :, 0], cache[:, :, 1]
    pages = torch.randperm(150, generator=torch.Generator().manual_seed(n)).int().to(gpu)
    table, free, prefix_table = pages[: 20 * batch].view(batch, 20).clone(), pages[20 * batch : 20 * batch + 30].clone(), pages[-20:][None].clone()
    lens, added, prefix_lens, cu_groups = i32(100, 40, 0), i32(*new), i32(310), i32(0, 2)
    q, k, v = (torch.empty(n, h, d, dtype=torch.bfloat16, device=gpu) for h in (heads, kv_heads, kv_heads))
    made = paged_cache_tables(lens, added, table.clone(), free, size, n)
    outs = [(torch.empty_like(q), torch.empty(heads, n, device=gpu)) for _ in range(2)]
    own = dict(cu_seqlens_q=made.cu_seqlens, max_seqlen_q=max(new), max_seqlen_k=300)
    own_args, prefix_args = (q, k_cache, v_cache, table, made.seq_lens), (q, k_cache, v_cache, prefix_table, prefix_lens, cu_groups, table, made.seq_lens)
    workspaces = [torch.empty(max(x, 1), dtype=torch.uint8, device=gpu) for x in (paged_cache_workspace_bytes(*own_args, **own),
                                                                                 shared_prefix_workspace_bytes(*prefix_args, **own))]

    def step():
        paged_cache_tables(lens, added, table, free, size, n, out=made)
        paged_cache_write(k, v, made.slot_mapping, k_cache, v_cache)
        paged_cache_attention(*own_args, **own, out=outs[0][0], lse=outs[0][1], workspace=workspaces[0])
        shared_prefix_attention(*prefix_args, **own, out=outs[1][0], lse=outs[1][1], workspace=workspaces[1])

    def fill(turn):
        lens.copy_(torch.tensor([[100, 40, 0], [3, 0, 17], [230, 200, 64]][turn % 3], dtype=torch.int32))
        prefix_lens.fill_([310, 17, 0][turn % 3])
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
            for t in (*outs[0], *outs[1], *made):
                t.fill_(7)
            torch.cuda.synchronize()
            if again:
                recording.run(0, 4, stream.cuda_stream)
            else:
                step()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (*state, *outs[0], *outs[1], *made)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), turn
        assert not torch.isnan(results[0][2]).any() and (results[0][2] != 7).any()
