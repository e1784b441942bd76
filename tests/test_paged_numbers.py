"""Numbers that the tables and writes of a paged cache do not hold are refused, not cut to 32 bits (CPU: nothing is launched)."""

import pytest
import torch

from dcp_amd.ops import paged_cache, paged_cache_tables, paged_cache_write


@pytest.fixture
def here(monkeypatch):
    """Tensors without memory on "the current device", and the calls that would have been made."""
    calls = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: torch.empty(0, device="meta").get_device())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0)
    monkeypatch.setattr(paged_cache._lib, "call", lambda *args: calls.append(args))
    return calls


def _empty(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


def _tables(page_size=16, n_tokens=4, n=2, width=3, free=5):
    return paged_cache_tables(_empty(n), _empty(n), _empty(n, width), _empty(free), page_size, n_tokens)


def _write(n_tokens=3, heads=2, head_dim=8, n_pages=4, page_size=16):
    x, cache = _empty(n_tokens, heads, head_dim, dtype=torch.uint8), _empty(n_pages, page_size, heads, head_dim, dtype=torch.uint8)
    paged_cache_write(x, x, _empty(n_tokens, dtype=torch.int64), cache, cache)


def test_numbers_that_fit(here):
    _tables(2**31 - 1, 2**31 - 1)
    _tables(16.0, torch.tensor(4))
    _write()
    _write(n_pages=2**33)  # (counted in 64 bits)
    assert [call[0] for call in here] == ["dcp_paged_cache_tables"] * 2 + ["dcp_paged_cache_write"] * 2
    assert here[0][-3:-1] == (2**31 - 1, 2**31 - 1) and here[1][-3:-1] == (16, 4) and here[3][12] == 2**33


@pytest.mark.parametrize("wrong", [dict(page_size=2**32 + 16), dict(page_size=2**31), dict(page_size=16.5), dict(n_tokens=2**32 + 4),
                                   dict(n_tokens=4.25), dict(n_tokens=-(2**32)), dict(page_size=float("nan")), dict(page_size=float("inf")),
                                   dict(width=2**32 + 3), dict(free=2**32 + 5), dict(n=2**32 + 2)])
def test_numbers_of_tables_that_do_not(here, wrong):
    with pytest.raises(ValueError, match="32 bits"):
        _tables(**wrong)
    assert not here


@pytest.mark.parametrize("wrong", [dict(n_tokens=2**32 + 3), dict(heads=2**32 + 2), dict(head_dim=2**32 + 8), dict(page_size=2**32 + 16)])
def test_sizes_of_writes_that_do_not(here, wrong):
    with pytest.raises(ValueError, match="32 bits"):
        _write(**wrong)
    assert not here


@pytest.mark.parametrize("scale", [1e39, -1e39, "half"])
def test_a_scale_that_32_bits_do_not_hold(here, scale):
    from dcp_amd.flash_attn_interface import _paged_args

    bf16 = torch.bfloat16
    q, cache = _empty(2, 4, 64, dtype=bf16), _empty(3, 16, 2, 64, dtype=bf16)
    with pytest.raises(ValueError, match="softmax_scale"):
        _paged_args(q, cache, cache, _empty(2, 3), _empty(2), None, None, None, scale, None, 0, None, None)
