"""Paged caches for the tests of the operators that answer over them, and those operators' definitions in 64 bits."""

import math

import numpy as np
import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative


class Paged:
    """Requests (and prefixes) with keys in a cache whose every other place holds NaN.  Built on the CPU from ``seed`` alone;
    ``to(device)`` moves the tensors that the operators take."""

    def __init__(self, keys, new=None, heads=8, kv_heads=2, head_dim=128, page_size=64, dtype=torch.bfloat16, window=0, n_starting=0,
                 prefixes=(), cu_groups=(), layout="halves", extra_tokens=0, extra_pages=2, bad=(), seed=0, q_scale=2.0):
        g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
        self.keys, self.new = list(keys), [1] * len(keys) if new is None else list(new)
        self.heads, self.kv_heads, self.head_dim, self.page_size, self.dtype = heads, kv_heads, head_dim, page_size, dtype
        self.window, self.n_starting, self.prefixes, self.cu_groups = window, n_starting, list(prefixes), list(cu_groups)
        rows = self.keys + self.prefixes
        counts = [-(-n // page_size) for n in rows]
        n_pages = sum(counts) + extra_pages
        pages, width = iter(rng.permutation(n_pages).tolist()), max(1, max(counts, default=1))
        table = np.full((len(rows), width), -1, dtype=np.int32)
        for i, n in enumerate(counts):
            table[i, :n] = [next(pages) for _ in range(n)]
        total = sum(self.new) + extra_tokens
        self.q = (torch.randn(total, heads, head_dim, generator=g) * q_scale).to(dtype)
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        shape = dict(halves=(n_pages, page_size, 2, kv_heads, head_dim), apart=(2, n_pages, page_size, kv_heads, head_dim),
                     by_head=(2, n_pages, kv_heads, page_size, head_dim))[layout]
        self.store = torch.full(shape, math.nan, dtype=dtype)
        k, v = self.caches(self.store, layout)
        self.layout, self.n_pages = layout, n_pages
        self.k_rows, self.v_rows = [], []
        for i, n in enumerate(rows):
            kr, vr = (torch.randn(n, kv_heads, head_dim, generator=g).to(dtype) for _ in range(2))
            self.k_rows.append(kr)
            self.v_rows.append(vr)
            j = np.arange(n)
            seen = np.ones(n, dtype=bool)
            if i < len(keys) and window:  # keys that no query of the request sees are left NaN
                seen = (j < n_starting) | (j > n - self.new[i] - window)
            j = j[seen]
            at, off = torch.as_tensor(table[i, j // page_size].astype(np.int64)), torch.as_tensor(j % page_size)
            k[at, off], v[at, off] = kr[seen], vr[seen]
        self.hidden = [set() for _ in rows]
        for i, column, entry in bad:  # table entries that name no page
            table[i, column] = entry(n_pages)
            self.hidden[i] = self.hidden[i] | set(range(column * page_size, (column + 1) * page_size))
        self.table, self.prefix_table = table[: len(keys)], table[len(keys):]

    @staticmethod
    def caches(store, layout):
        if layout == "halves":
            return store[:, :, 0], store[:, :, 1]
        return (store[0], store[1]) if layout == "apart" else (store[0].transpose(1, 2), store[1].transpose(1, 2))

    def to(self, device):
        i32 = lambda x: torch.as_tensor(np.asarray(x, dtype=np.int32), device=device)
        k, v = self.caches(self.store.to(device), self.layout)
        made = dict(q=self.q.to(device), k_cache=k, v_cache=v, block_table=i32(self.table), seq_lens=i32(self.keys))
        if any(n != 1 for n in self.new) or len(self.q) != len(self.new):
            made.update(cu_seqlens_q=i32(self.cu), max_seqlen_q=max(self.new))
        if self.prefixes:
            made.update(prefix_table=i32(self.prefix_table), prefix_lens=i32(self.prefixes), cu_groups=i32(self.cu_groups))
        elif self.window:
            made.update(window=self.window, n_starting=self.n_starting)
        return made

    def truth(self):
        """``out``, ``lse`` in 64 bits and how far a kernel may be off each of them, NaN for tokens of no request.

        The bounds: a product of D terms and a sum of N in 32 bits are off by at most D resp. N steps of 2^-23 relative to the sum of
        their terms' sizes (each operation by one; the matrix instructions' rounding is not stated, so a step, not half a step).  A
        score off by d makes its weight off by a factor exp(d), so the weighted sum and the sum of the weights by 2 d together.  The
        weights are rounded to the storage type (half a step, or 2^-25 where fp16 has no normal number; the largest
        weight is at least 1 before the division), the result once more."""
        u, step, scale, group = U[self.dtype], 2.0**-23, self.head_dim**-0.5, self.heads // self.kv_heads
        total = len(self.q)
        out = torch.full((total, self.heads, self.head_dim), math.nan, dtype=torch.float64)
        lse = torch.full((self.heads, total), math.nan, dtype=torch.float64)
        out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
        for b, (n, new) in enumerate(zip(self.keys, self.new)):
            sources = [(self.k_rows[b], self.v_rows[b], self.hidden[b], False)]
            for i in range(len(self.prefixes)):
                if self.cu_groups[i] <= b < self.cu_groups[i + 1]:
                    at = len(self.keys) + i
                    sources.append((self.k_rows[at], self.v_rows[at], self.hidden[at], True))
            k, v = (torch.cat([s[x] for s in sources]).double() for x in (0, 1))
            x = torch.arange(n - new, n)[:, None]
            visible = []
            for kr, _, hidden, is_prefix in sources:
                j = torch.arange(len(kr))
                see = torch.ones(new, len(kr), dtype=torch.bool) if is_prefix else j <= x
                if self.window and not is_prefix:
                    see = see & ((j < self.n_starting) | (j > x - self.window))
                see[:, [p for p in hidden if p < len(kr)]] = False
                visible.append(see)
            visible = torch.cat(visible, 1)
            rows = slice(int(self.cu[b]), int(self.cu[b]) + new)
            for h in range(self.heads):
                q, kh, vh = self.q[rows, h].double(), k[:, h // group], v[:, h // group]
                s = (q @ kh.t() * scale).masked_fill(~visible, -math.inf)
                some = visible.any(1)
                total_lse = torch.logsumexp(s, 1) if s.shape[1] else torch.full((new,), -math.inf, dtype=torch.float64)
                p = torch.where(some[:, None], torch.exp(s - torch.where(some, total_lse, 0.0)[:, None]), 0.0)
                sizes = (q.abs() @ kh.abs().t() * scale).masked_fill(~visible, 0.0)
                # (the exponent's argument has two roundings of numbers no larger than the scores, the exponential two steps of its own)
                off = (sizes.amax(1) if s.shape[1] else torch.zeros(new, dtype=torch.float64)) * (self.head_dim + 4) * step + 2 * step
                count = visible.sum(1) + 256  # (and the joining of shares)
                o, a = p @ vh, p @ vh.abs()
                tiny = (visible.double() @ vh.abs()) * 2.0**-25 if self.dtype is torch.float16 else 0.0
                out[rows, h], lse[h, rows] = o, torch.where(some, total_lse, math.inf)
                out_tol[rows, h] = u * (1 + 2 * u) * (a + o.abs()) + a * (2 * off + 2 * count * step)[:, None] + tiny + 2.0**-25 * (self.dtype is torch.float16)
                lse_tol[h, rows] = off + count * step + torch.where(some, total_lse.abs(), 0.0) * 4 * step
        return out, lse, out_tol, lse_tol


def check(got, truth, untouched=None):
    """``got``: (out, lse) of the device; ``untouched``: what tokens of no request hold."""
    out, lse = (t.double().cpu() for t in got)
    want_out, want_lse, out_tol, lse_tol = truth
    ours = ~torch.isnan(want_lse[0])
    for name, x, y, tol in (("out", out[ours], want_out[ours], out_tol[ours]), ("lse", lse[:, ours], want_lse[:, ours], lse_tol[:, ours])):
        assert not torch.isnan(x).any(), f"{name}: {int(torch.isnan(x).sum())} NaN"
        assert torch.equal(torch.isinf(x), torch.isinf(y)), f"{name}: infinities"
        off = torch.where(torch.isinf(y), 0.0, (x - torch.where(torch.isinf(y), x, y)).abs() - tol)
        assert off.numel() == 0 or off.max() <= 0, f"{name}: {off.max():.3g} over the bound at {np.unravel_index(int(off.argmax()), off.shape)}"
    if untouched is not None:
        assert (out[~ours] == untouched).all() and (lse[:, ~ours] == untouched).all(), "tokens of no request were written"


def tables_truth(cached, new, table, free, page_size, n_tokens):
    """``paged_cache_tables`` token by token."""
    table, taken, slots, positions, cu = table.copy(), 0, [], [], [0]
    width = table.shape[1]
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        have, want = min(-(-c // page_size), width), min(-(-(c + n) // page_size), width)
        for i in range(have, want):
            table[b, i] = free[taken] if taken < len(free) else -1
            taken += 1
        for x in range(c, c + n):
            page = table[b, x // page_size] if x // page_size < width else -1
            slots.append(int(page) * page_size + x % page_size if page >= 0 else -1)
            positions.append(x)
        cu.append(cu[-1] + n)
    pad = max(0, n_tokens - len(slots))
    return dict(slot_mapping=(slots + [-1] * pad)[:n_tokens], positions=(positions + [0] * pad)[:n_tokens], cu_seqlens=cu,
                seq_lens=[max(c, 0) + max(n, 0) for c, n in zip(cached, new)], pages_taken=[taken]), table
