"""A paged K/V cache held in 4 bits: its pages, writes into it through the slots of ``paged_cache_tables``, and rows taken back to
16 bits.  ``dcp_amd.flash_attn_interface.quantized_cache_attention`` answers over it.

Every 32 neighbouring elements of a token's key or value share a power of two, and each is one of 16 numbers times that:
+-{0, 0.5, 1, 1.5, 2, 3, 4, 6}.  That is 17/32 of a byte an element, 3.8 times fewer than 16 bits.

Work is enqueued on torch's current stream; nothing waits for the device, so a step may be captured into a graph.
There is no fallback: without the built library these raise.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from dcp_amd import _lib
from dcp_amd.ops.fused_ops import dtype_code
from dcp_amd.ops.paged_cache import _check, _in_32_bits

__all__ = ["quantized_cache_pages", "quantized_cache_read", "quantized_cache_write"]


def quantized_cache_pages(n_pages: int, page_size: int, n_heads_kv: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Pages of zeros for keys and values of this shape: uint8 ``[n_pages, n_heads_kv, page_size // 16, 17 * head_dim]``, the
    bytes of 16 tokens of a head together (``dcp_hip.h`` has their order).  Page sizes are multiples of 16, head sizes 64 or 128."""
    if page_size < 1 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    return torch.zeros(n_pages, n_heads_kv, page_size // 16, 17 * head_dim, dtype=torch.uint8, device=device)


# A short call is as long as its checks and its launch (3 of 6 us), so what is as it should be passes in one expression; what is not is told
# apart afterwards.
def _cache_args(cache: torch.Tensor, here: int) -> tuple:
    """``(address, heads, head size, pages, page size, page stride, head stride)`` of a cache on the current device."""
    try:
        shape, strides = cache.shape, cache.stride()
        good = (len(shape) == 4 and (shape[3] == 2176 or shape[3] == 1088) and strides[3] == 1 and shape[2] > 0 and
                (strides[2] == shape[3] or shape[2] == 1) and cache.dtype is torch.uint8 and cache.get_device() == here)
    except AttributeError:
        good = False
    if not good:
        _check(cache, torch.uint8, "cache", here, dense=False)
        raise ValueError("cache must be [n_pages, n_heads_kv, page_size // 16, 17 * head_dim] of head size 64 or 128, dense in the "
                         f"last two, got {list(shape)} with strides {list(strides)}")
    return cache.data_ptr(), shape[1], shape[3] // 17, shape[0], 16 * shape[2], strides[0], strides[1]


def _rows(k, v, slot_mapping, heads: int, head_dim: int, here: int) -> tuple:
    """``(k, v, slots, n_tokens, dtype, token stride, head stride, v's two)`` of rows that belong into a cache of these sizes; the last is None
    where v has the strides of k."""
    try:
        dtype, shape, strides = k.dtype, k.shape, k.stride()
        good = (len(shape) == 3 and shape[1] == heads and shape[2] == head_dim and strides[2] == 1 and shape == v.shape and strides == v.stride() and
                v.dtype is dtype and k.get_device() == here and v.get_device() == here and
                slot_mapping.dtype is torch.int64 and slot_mapping.dim() == 1 and slot_mapping.get_device() == here and
                slot_mapping.is_contiguous() and slot_mapping.shape[0] == shape[0])
    except AttributeError:
        good, dtype = False, getattr(k, "dtype", torch.bfloat16)
    v_strides = None
    if not good:
        _check(k, dtype, "k", here, dense=False), _check(v, dtype, "v", here, dense=False)
        if k.dim() != 3 or tuple(k.shape[1:]) != (heads, head_dim) or k.shape != v.shape or k.stride(2) != 1 or v.stride(2) != 1:
            raise ValueError(f"k and v must be [n_tokens, {heads}, {head_dim}] with dense rows, got {list(k.shape)} and {list(v.shape)}")
        _check(slot_mapping, torch.int64, "slot_mapping", here, (k.shape[0],))
        v_strides = v.stride()[:2]
    return k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(), shape[0], dtype_code(dtype), strides[0], strides[1], v_strides


def quantized_cache_write(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, cache: torch.Tensor) -> None:
    """Writes ``k`` and ``v`` (bf16 or fp16 ``[n_tokens, n_heads_kv, D]``, each at any strides that are multiples of 8) into ``cache``
    (``quantized_cache_pages``) at ``slot_mapping`` (int64 ``[n_tokens]``: ``page * page_size + offset``).

    A block of 32 elements takes the smallest power of two 2^e of which none of them is more than 7 times as large, an element the
    nearest of the numbers there are, ties to the even code: it is off by at most 2^e, by 2^e / 4 where it is below 2^(e + 1).  (A block
    with one of the type's largest numbers takes those that the type holds, and may be off by a quarter of its largest.)  A block with
    an infinity or a NaN reads as NaN.  Slots outside of the cache are skipped, so the -1 of padding writes nothing; the others
    have to differ from each other, and ``k`` and ``v`` may not lie in the cache."""
    here = torch._C._cuda_getDevice()
    cache_at, heads, head_dim, n_pages, page_size, page, head = _cache_args(cache, here)
    k_at, v_at, slots, n_tokens, dtype, token_stride, head_stride, v_strides = _rows(k, v, slot_mapping, heads, head_dim, here)
    if (n_tokens | page_size | heads) >> 31:
        _in_32_bits(n_tokens=n_tokens, page_size=page_size, n_heads_kv=heads)
    if v_strides is None:
        _lib.call("dcp_quantized_cache_write", k_at, v_at, slots, cache_at, n_tokens, heads, head_dim, dtype, token_stride, head_stride, n_pages,
                  page_size, page, head, torch._C._cuda_getCurrentRawStream(here))
    else:
        _lib.call("dcp_quantized_cache_write_strided", k_at, v_at, slots, cache_at, n_tokens, heads, head_dim, dtype, token_stride, head_stride,
                  *v_strides, n_pages, page_size, page, head, torch._C._cuda_getCurrentRawStream(here))


def quantized_cache_read(cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                         out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows at ``slot_mapping`` (int64 ``[n_tokens]``) as ``(k, v)``, ``[n_tokens, n_heads_kv, D]`` of ``dtype`` (bf16 or fp16):
    what ``quantized_cache_attention`` sees of them.  Rows written from this type are exact; what the type does not hold is rounded.
    Rows of slots outside of the cache are zeros.  ``out``: two tensors to write to, not in the cache (``dtype`` is then theirs);
    each at any strides that are multiples of 8 and put no two rows at the same place."""
    here = torch._C._cuda_getDevice()
    cache_at, heads, head_dim, n_pages, page_size, page, head = _cache_args(cache, here)
    if out is None:
        _check(slot_mapping, torch.int64, "slot_mapping", here)
        if slot_mapping.dim() != 1:
            raise ValueError(f"slot_mapping must have one axis, got {list(slot_mapping.shape)}")
        n_tokens, code = slot_mapping.shape[0], dtype_code(dtype)
        k = cache.new_empty((n_tokens, heads, head_dim), dtype=dtype)
        v = torch.empty_like(k)
        k_at, v_at, slots, token_stride, head_stride = k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(), heads * head_dim, head_dim
        v_strides = None
    else:
        k, v = out
        k_at, v_at, slots, n_tokens, code, token_stride, head_stride, v_strides = _rows(k, v, slot_mapping, heads, head_dim, here)
    if (n_tokens | page_size | heads) >> 31:
        _in_32_bits(n_tokens=n_tokens, page_size=page_size, n_heads_kv=heads)
    if v_strides is None:
        _lib.call("dcp_quantized_cache_read", cache_at, slots, k_at, v_at, n_tokens, heads, head_dim, code, token_stride, head_stride, n_pages,
                  page_size, page, head, torch._C._cuda_getCurrentRawStream(here))
    else:
        _lib.call("dcp_quantized_cache_read_strided", cache_at, slots, k_at, v_at, n_tokens, heads, head_dim, code, token_stride, head_stride,
                  *v_strides, n_pages, page_size, page, head, torch._C._cuda_getCurrentRawStream(here))
    return k, v
