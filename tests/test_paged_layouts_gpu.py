"""Paged attention by several kv heads a workgroup, and own keys and prefixes whose cases share a name, against 64 bits."""

import pytest
import torch

from dcp_amd.flash_attn_interface import (paged_cache_attention, paged_cache_workspace_bytes, shared_prefix_attention,
                                          shared_prefix_workspace_bytes)
from tests.paged_cases import Paged, check
from tests.test_paged_attention_gpu import PREFIXES, SINGLE

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _cut_bytes(case, heads, rows):
    """Where the pieces of rows are, and two pieces a workgroup of ``heads`` kv heads of ``rows`` rows, two workgroups a CU."""
    workgroups, queries = 2 * torch.cuda.get_device_properties(0).multi_processor_count, len(case.q) * case.heads
    return (queries * 8 + 15) // 16 * 16 + workgroups * 2 * heads * rows * (case.head_dim + 2) * 4


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("new,rows", [(None, 16), ([8, 1, 5, 0, 3], 32)])
@pytest.mark.parametrize("kv_heads,heads", [(2, 2), (4, 4), (6, 2), (8, 4)])
@pytest.mark.parametrize("head_dim,dtype", [(128, torch.bfloat16), (64, F16)])
def test_equal_shares_of_several_heads(gpu, head_dim, dtype, kv_heads, heads, new, rows, prefix):
    """Told of long keys, the host deals shares of two or four heads at once; requests that are short are cut all the same."""
    more = dict(prefixes=[300, 70], cu_groups=[0, 2, 4]) if prefix else {}
    case = Paged([1000, 3, 517, 0, 64], new=new, heads=4 * kv_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=16, dtype=dtype, **more)
    args = dict(case.to(gpu), max_seqlen_k=1 << 20)
    n = (shared_prefix_workspace_bytes if prefix else paged_cache_workspace_bytes)(**args)
    shares, share = n - _cut_bytes(case, heads, rows), len(case.q) * case.heads * (head_dim + 2) * 4
    # (odd numbers of tokens: no share of all rows is as large as a power of two of pieces)
    assert len(case.q) % 2 == 1 and (shares >= 2 * share and shares % share == 0 if prefix else shares == 0)
    store = torch.full((n + 4096,), 0xEE, dtype=torch.uint8, device=gpu)
    got = (shared_prefix_attention if prefix else paged_cache_attention)(**args, workspace=store[:n])
    check(got, case.truth())
    assert (store[n:] == 0xEE).all()


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("kv_heads,heads", [(2, 2), (4, 4), (8, 4)])
def test_shares_of_several_heads_that_hold_several_requests(gpu, kv_heads, heads, prefix):
    """More turns than workgroups: shares begin and end in the middle of requests and pass over others."""
    more = dict(prefixes=[200], cu_groups=[50, 150]) if prefix else {}
    case = Paged([(37 * i) % 211 for i in range(251)], heads=kv_heads, kv_heads=kv_heads, head_dim=64, page_size=16, **more)
    args = dict(case.to(gpu), max_seqlen_k=1 << 20)
    n = (shared_prefix_workspace_bytes if prefix else paged_cache_workspace_bytes)(**args)
    assert n >= _cut_bytes(case, heads, 16) and (prefix or n == _cut_bytes(case, heads, 16))
    check((shared_prefix_attention if prefix else paged_cache_attention)(**args), case.truth())


@pytest.mark.parametrize("more", [{}, dict(window=20, n_starting=3), dict(prefixes=[100, 33], cu_groups=[3, 200, 280])],
                         ids=["causal", "window", "prefix"])
@pytest.mark.parametrize("kv_heads", [2, 4, 6])  # (two, four and two heads: 600 units and more for 512 workgroups)
@pytest.mark.parametrize("many_tokens", [False, True])
@pytest.mark.parametrize("head_dim,dtype", [(128, torch.bfloat16), (64, F16)])
def test_whole_units_of_several_heads(gpu, head_dim, dtype, many_tokens, kv_heads, more):
    new = [(1, 0, 9, 4, 16)[i % 5] for i in range(300)] if many_tokens else None
    case = Paged([(i * 7) % 65 for i in range(300)], new=new, heads=2 * kv_heads, kv_heads=kv_heads, head_dim=head_dim, page_size=16, dtype=dtype,
                 **more)
    args = dict(case.to(gpu), max_seqlen_k=64)
    if not more.get("prefixes"):
        assert paged_cache_workspace_bytes(**args) == 0
    check((shared_prefix_attention if case.prefixes else paged_cache_attention)(**args), case.truth())


@pytest.mark.parametrize("longest_q", [1, 5, 1000])
@pytest.mark.parametrize("cases,name", [(SINGLE, "many"), (SINGLE, "fp16_d64"), (SINGLE, "group_5"), (PREFIXES, "many"), (PREFIXES, "fp16_d64"),
                                        (PREFIXES, "group_5")], ids=lambda x: x if isinstance(x, str) else "prefix" if x is PREFIXES else "own")
def test_numbers_of_tokens_the_host_does_not_know(gpu, cases, name, longest_q):
    case = Paged(**cases[name])
    args = {**case.to(gpu), "cu_seqlens_q": torch.tensor(case.cu, dtype=torch.int32, device=gpu), "max_seqlen_q": longest_q}
    check((shared_prefix_attention if case.prefixes else paged_cache_attention)(**args), case.truth())


@pytest.mark.parametrize("longest", [64, 700, 5000, 1 << 20])
@pytest.mark.parametrize("cases,name", [(SINGLE, "many"), (SINGLE, "fp16_d64"), (SINGLE, "group_5"), (PREFIXES, "many"), (PREFIXES, "fp16_d64"),
                                        (PREFIXES, "group_5")], ids=lambda x: x if isinstance(x, str) else "prefix" if x is PREFIXES else "own")
def test_units_whole_and_cut(gpu, cases, name, longest):
    case = Paged(**cases[name])
    check((shared_prefix_attention if case.prefixes else paged_cache_attention)(**case.to(gpu), max_seqlen_k=longest), case.truth())
