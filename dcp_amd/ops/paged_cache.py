"""The tables of a paged K/V cache and the writes through them: what a step of answering needs beside
``dcp_amd.flash_attn_interface.paged_cache_attention``.

Work is enqueued on torch's current stream; nothing waits for the device, so a step may be captured into a graph.
There is no fallback: without the built library these raise.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from dcp_amd import _lib
from dcp_amd.ops.fused_ops import _stream

__all__ = ["PagedCacheTables", "paged_cache_tables", "paged_cache_write"]


class PagedCacheTables(NamedTuple):
    """One step's tables (``paged_cache_tables``)."""

    slot_mapping: torch.Tensor  # int64 [n_tokens]: page * page_size + offset of every new token, -1 for none
    positions: torch.Tensor  # int32 [n_tokens]: its place in its request
    cu_seqlens: torch.Tensor  # int32 [B + 1]: sums of the new tokens
    seq_lens: torch.Tensor  # int32 [B]: tokens of the requests, the new ones among them
    pages_taken: torch.Tensor  # int32 [1]


def _here(t, dtype, name: str, shape=None, dense: bool = True) -> int:
    """The address of a tensor of the current device with this type (and, if given, this shape)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name} must be a tensor of the current device")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


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
    write to.
    """
    n = cached_lens.shape[0] if isinstance(cached_lens, torch.Tensor) and cached_lens.dim() == 1 else -1
    i32 = torch.int32
    lens, new = _here(cached_lens, i32, "cached_lens", (n,)), _here(new_lens, i32, "new_lens", (n,))
    table = _here(block_table, i32, "block_table", dense=False)
    if block_table.dim() != 2 or block_table.shape[0] != n or block_table.shape[1] < 1 \
            or (n > 0 and block_table.shape[1] > 1 and block_table.stride(1) != 1) or (n > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError(f"block_table must be [{n}, pages] with dense rows, got {list(block_table.shape)}")
    free = _here(free_pages, i32, "free_pages")
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must have one axis, got {list(free_pages.shape)}")
    n_tokens = int(n_tokens)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    if out is None:
        device = cached_lens.device
        out = PagedCacheTables(torch.empty(n_tokens, dtype=torch.int64, device=device), torch.empty(n_tokens, dtype=i32, device=device),
                               torch.empty(n + 1, dtype=i32, device=device), torch.empty(n, dtype=i32, device=device),
                               torch.empty(1, dtype=i32, device=device))
    _lib.call("dcp_paged_cache_tables", lens, new, table, max(block_table.stride(0), block_table.shape[1]), free,
              _here(out.slot_mapping, torch.int64, "slot_mapping", (n_tokens,)), _here(out.positions, i32, "positions", (n_tokens,)),
              _here(out.cu_seqlens, i32, "cu_seqlens", (n + 1,)), _here(out.seq_lens, i32, "seq_lens", (n,)),
              _here(out.pages_taken, i32, "pages_taken", (1,)), n, block_table.shape[1], free_pages.shape[0], int(page_size),
              n_tokens, _stream())
    return out


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    """Writes ``k`` and ``v`` (``[n_tokens, n_heads_kv, D]``) into the caches (``[n_pages, page_size, n_heads_kv, D]``, any
    strides, a cache's two halves for instance) at ``slot_mapping`` (int64 ``[n_tokens]``).  Slots outside of the cache are skipped,
    so the -1 of padding writes nothing; the others have to differ from each other.  Any type of 1, 2 or 4 bytes."""
    dtype = k_cache.dtype
    addresses = [_here(t, dtype, name, dense=False) for t, name in ((k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"))]
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
        raise ValueError("k_cache and v_cache must be [n_pages, page_size, n_heads_kv, D] with the same strides and dense rows")
    n_pages, page_size, heads, head_dim = k_cache.shape
    if k.dim() != 3 or k.shape != v.shape or k.stride() != v.stride() or tuple(k.shape[1:]) != (heads, head_dim) or (head_dim > 1 and k.stride(2) != 1):
        raise ValueError(f"k and v must be [n_tokens, {heads}, {head_dim}] with the same strides and dense rows")
    slots = _here(slot_mapping, torch.int64, "slot_mapping", (k.shape[0],))
    _lib.call("dcp_paged_cache_write", addresses[0], addresses[1], slots, addresses[2], addresses[3], k.shape[0], heads, head_dim,
              k.element_size(), k.stride(0), k.stride(1), n_pages, page_size, k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
              _stream())
