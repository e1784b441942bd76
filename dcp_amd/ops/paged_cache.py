"""The tables of a paged K/V cache and the writes through them: what a step of answering needs beside
``dcp_amd.flash_attn_interface.paged_cache_attention``.

Work is enqueued on torch's current stream; nothing waits for the device, so a step may be captured into a graph.
There is no fallback: without the built library these raise.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from dcp_amd import _lib

__all__ = ["PagedCacheTables", "paged_cache_tables", "paged_cache_write"]


class PagedCacheTables(NamedTuple):
    """One step's tables (``paged_cache_tables``)."""

    slot_mapping: torch.Tensor  # int64 [n_tokens]: page * page_size + offset of every new token, -1 for none
    positions: torch.Tensor  # int32 [n_tokens]: its place in its request
    cu_seqlens: torch.Tensor  # int32 [B + 1]: sums of the new tokens
    seq_lens: torch.Tensor  # int32 [B]: tokens of the requests, the new ones among them
    pages_taken: torch.Tensor  # int32 [1]


def _check(t, dtype, name: str, here: int, shape=None, dense: bool = True) -> int:
    """The address of a tensor of this type on the current device (``here``), with this shape if one is given."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != here:
        raise ValueError(f"{name} must be a tensor of the current device")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _in_32_bits(**numbers) -> list:
    """The numbers as whole ones of 32 bits, which is what the library takes: the call would cut any other without a word."""
    for name, x in numbers.items():
        if not -(2**31) <= x < 2**31 or int(x) != x:
            raise ValueError(f"{name} must be a whole number of 32 bits, got {x}")
    return [int(x) for x in numbers.values()]


def paged_cache_tables(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                       page_size: int, n_tokens: int, out: Optional[PagedCacheTables] = None) -> PagedCacheTables:
    """The tables of a step in which request ``b``, with ``cached_lens[b]`` tokens in the cache, adds ``new_lens[b]``.

    Takes the pages the new tokens need from ``free_pages``, in order, appends them to the rows of ``block_table``
    (int32 ``[B, W]``, in place; entries behind a row's last page are left as they were) and returns a slot and a position
    for every new token.  ``n_tokens`` is the length of the token tables: at least the sum of ``new_lens``, which the
    caller knows on the host or bounds (tokens behind the last request's get slot -1 and position 0; those that do not
    fit are not entered).  ``pages_taken`` says how many pages the step takes: where that is more than there are,
    the missing ones are entered as -1 and their tokens get slot -1, as do tokens past ``W`` pages.  ``free_pages`` itself is
    not changed: drop its first ``pages_taken`` entries for the next step.  ``out``: tables of an earlier call to
    write to, none of which may be an input (the last step's ``seq_lens`` as ``cached_lens``: copy them first).
    """
    here, i32 = torch._C._cuda_getDevice(), torch.int32
    n = cached_lens.shape[0] if isinstance(cached_lens, torch.Tensor) and cached_lens.dim() == 1 else -1
    lens, new = _check(cached_lens, i32, "cached_lens", here, (n,)), _check(new_lens, i32, "new_lens", here, (n,))
    table = _check(block_table, i32, "block_table", here, dense=False)
    rows, width = block_table.shape if block_table.dim() == 2 else (-1, 0)
    stride = block_table.stride(0) if rows > 1 else width
    if rows != n or width < 1 or (n > 0 and width > 1 and block_table.stride(1) != 1) or (n > 1 and stride < width):
        raise ValueError(f"block_table must be [{n}, pages] with dense rows, got {list(block_table.shape)}")
    free = _check(free_pages, i32, "free_pages", here)
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must have one axis, got {list(free_pages.shape)}")
    n_free = free_pages.shape[0]
    # (asked in one question of sizes that are right: number by number this is 0.4 us of the call's ten)
    if type(n_tokens) is not int or type(page_size) is not int or (n_tokens | page_size | n | width | n_free) >> 31:
        n_tokens, page_size, *_ = _in_32_bits(n_tokens=n_tokens, page_size=page_size, B=n, pages=width, n_free=n_free)
        if n_tokens < 0:
            raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    if out is None:  # (one tensor for the four of 32 bits: five allocations are a third of a small step's time)
        ints = cached_lens.new_empty(n_tokens + 2 * n + 2)
        positions, cu, lens_out, taken = ints.split_with_sizes([n_tokens, n + 1, n, 1])
        out = PagedCacheTables(torch.empty(n_tokens, dtype=torch.int64, device=cached_lens.device), positions, cu, lens_out, taken)
        at = ints.data_ptr()
        addresses = (out.slot_mapping.data_ptr(), at, at + 4 * n_tokens, at + 4 * (n_tokens + n + 1), at + 4 * (n_tokens + 2 * n + 1))
    else:
        addresses = (_check(out.slot_mapping, torch.int64, "slot_mapping", here, (n_tokens,)),
                     _check(out.positions, i32, "positions", here, (n_tokens,)), _check(out.cu_seqlens, i32, "cu_seqlens", here, (n + 1,)),
                     _check(out.seq_lens, i32, "seq_lens", here, (n,)), _check(out.pages_taken, i32, "pages_taken", here, (1,)))
    _lib.call("dcp_paged_cache_tables", lens, new, table, stride, free, *addresses, n, width, n_free, page_size, n_tokens,
              torch._C._cuda_getCurrentRawStream(here))
    return out


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    """Writes ``k`` and ``v`` (``[n_tokens, n_heads_kv, D]``) into the caches (``[n_pages, page_size, n_heads_kv, D]``, any
    strides, a cache's two halves for instance) at ``slot_mapping`` (int64 ``[n_tokens]``).  Slots outside of the cache are skipped,
    so the -1 of padding writes nothing; the others have to differ from each other, and ``k`` and ``v`` may not lie in the caches.
    Any type of 1, 2 or 4 bytes."""
    here, dtype = torch._C._cuda_getDevice(), k_cache.dtype
    k_at, v_at = _check(k, dtype, "k", here, dense=False), _check(v, dtype, "v", here, dense=False)
    k_cache_at, v_cache_at = _check(k_cache, dtype, "k_cache", here, dense=False), _check(v_cache, dtype, "v_cache", here, dense=False)
    strides, in_strides = k_cache.stride(), k.stride()
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or strides != v_cache.stride() or strides[3] != 1:
        raise ValueError("k_cache and v_cache must be [n_pages, page_size, n_heads_kv, D] with the same strides and dense rows")
    n_pages, page_size, heads, head_dim = k_cache.shape
    if k.dim() != 3 or k.shape != v.shape or in_strides != v.stride() or tuple(k.shape[1:]) != (heads, head_dim) or (head_dim > 1 and in_strides[2] != 1):
        raise ValueError(f"k and v must be [n_tokens, {heads}, {head_dim}] with the same strides and dense rows")
    n_tokens = k.shape[0]
    if (n_tokens | page_size | heads | head_dim) >> 31:
        _in_32_bits(n_tokens=n_tokens, page_size=page_size, n_heads_kv=heads, D=head_dim)
    slots = _check(slot_mapping, torch.int64, "slot_mapping", here, (n_tokens,))
    _lib.call("dcp_paged_cache_write", k_at, v_at, slots, k_cache_at, v_cache_at, n_tokens, heads, head_dim, k.element_size(), in_strides[0],
              in_strides[1], n_pages, page_size, strides[0], strides[1], strides[2], torch._C._cuda_getCurrentRawStream(here))
