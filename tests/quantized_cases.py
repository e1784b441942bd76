"""A paged cache held in 4 bits for the tests of the operators that write, read and answer over it: its definition in 64 bits and byte by
byte."""

import functools

import numpy as np
import torch

from tests.paged_cases import Paged

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LARGEST = {torch.bfloat16: torch.finfo(torch.bfloat16).max, torch.float16: torch.finfo(torch.float16).max}


def quantize(x):
    """Codes and exponents' bytes of rows ``[..., D]`` of a 16-bit type, in 64 bits."""
    rows = x.double().numpy().reshape(-1, 32)
    finite = np.isfinite(rows).all(1)
    rows = np.where(finite[:, None], rows, 0.0)
    top = np.abs(rows).max(1, initial=0.0)
    e = np.where(top > 0, np.maximum(np.floor(np.log2(np.maximum(top, 1e-300))) - 4, -127), -127).astype(np.int64)
    while (more := top > 7 * 2.0 ** e.astype(float)).any():
        e += more
    scale = 2.0 ** e[:, None].astype(float)
    off = np.abs(np.abs(rows)[..., None] - LEVELS * scale[..., None])
    off[np.broadcast_to(LEVELS * scale[..., None] > LARGEST[x.dtype], off.shape)] = np.inf
    # the nearest, of two the one of even code
    best = np.where(off == off.min(-1, keepdims=True), 1 + (np.arange(8) % 2 == 0), 0).argmax(-1)
    codes = (best + 8 * np.signbit(rows)).astype(np.uint8)
    exponents = np.where(finite, e + 127, 255).astype(np.uint8)
    return codes.reshape(x.shape), exponents.reshape(*x.shape[:-1], x.shape[-1] // 32)


def values(codes, exponents):
    """The numbers in 64 bits."""
    e = np.repeat(exponents.astype(np.int64), 32, axis=-1)
    x = np.where(codes > 7, -1.0, 1.0) * LEVELS[codes & 7] * 2.0 ** (e - 127.0)
    return torch.from_numpy(np.where(e == 255, np.nan, x))


@functools.cache
def _bytes_of(d, j, of_v):
    """Where the bytes of codes and of exponents of token ``j`` of 16 are."""
    i, block = np.arange(d // 2), np.arange(d // 32)
    if not of_v:
        return j * (d // 2) + i, 16 * d + j * (d // 32) + block
    piece, in_piece = np.divmod(i, d // 32)
    return 8 * d + ((j // 4 * 16 + piece) * 4 + j % 4) * (d // 32) + in_piece, 16 * d + d // 2 + (j // 4 * (d // 32) + block) * 4 + j % 4


def put_row(tiles, j, of_v, codes, exponents):
    """Codes ``[heads, D]`` and exponents ``[heads, D / 32]`` of token ``j`` of 16 into their bytes ``tiles [heads, 17 D]``."""
    at, exponents_at = _bytes_of(codes.shape[1], j, bool(of_v))
    tiles[:, at] = codes[:, 0::2] | codes[:, 1::2] << 4
    tiles[:, exponents_at] = exponents


class Quantized(Paged):
    """``Paged`` with its keys and values in 4 bits.  Bytes of places that no query of their request sees are 0xff: codes of the largest
    size and no numbers."""

    def __init__(self, *args, **more):
        super().__init__(*args, **{**more, "layout": "halves"})
        d, size, kv = self.head_dim, self.page_size, self.store.numpy(force=True) if self.dtype != torch.bfloat16 else self.store.float().numpy()
        self.cache = np.full((self.n_pages, self.kv_heads, size // 16, 17 * d), 0xFF, dtype=np.uint8)
        for i, table_row in enumerate([*self.table, *self.prefix_table]):
            rows = []
            for of_v, kept in enumerate((self.k_rows[i], self.v_rows[i])):
                codes, exponents = quantize(kept)
                rows.append(values(codes, exponents).to(self.dtype))
                for j in range(len(kept)):
                    page, offset = int(table_row[j // size]), j % size
                    if not 0 <= page < self.n_pages or np.isnan(kv[page, offset]).all():
                        continue  # of no page, or seen by nobody
                    put_row(self.cache[page, :, offset // 16], offset % 16, of_v, codes[j], exponents[j])
            self.k_rows[i], self.v_rows[i] = rows
        self.cache = torch.from_numpy(self.cache)

    def to(self, device):
        made = super().to(device)
        del made["k_cache"], made["v_cache"]
        made["cache"] = self.cache.to(device)
        return made
