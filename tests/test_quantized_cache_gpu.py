"""Writes into a paged cache held in 4 bits and reads out of it on the GPU: byte by byte against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from dcp_amd.flash_attn_interface import quantized_cache_attention
from dcp_amd.ops import paged_cache_tables, quantized_cache_pages, quantized_cache_read, quantized_cache_write
from tests.quantized_cases import put_row, quantize, values

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _rows(n, heads, d, dtype, seed):
    """Rows of every size that the type has, with ties, zeros and negative zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g) * 2.0 ** torch.randint(-12, 12, (n, heads, 1), generator=g)
    kind = torch.randint(0, 6, (n, heads, 1), generator=g)
    x = torch.where(kind == 1, torch.randint(-28, 29, x.shape, generator=g) * 0.25, x)
    x = torch.where(kind == 2, x * (torch.rand(x.shape, generator=g) < 0.05), x)
    return x.to(dtype)


def _written(cache, slots, k, v, page_size):
    """``cache`` (numpy) after a write."""
    for of_v, x in enumerate((k, v)):
        codes, exponents = quantize(x)
        for t, slot in enumerate(slots):
            if 0 <= slot < cache.shape[0] * page_size:
                page, offset = divmod(slot, page_size)
                put_row(cache[page, :, offset // 16], offset % 16, of_v, codes[t], exponents[t])
    return cache


def _same_bytes(got, want, d):
    """Equal but for the sign of a zero, whose code is 0 or 8."""
    got, want = got.astype(np.int32), want.astype(np.int32)
    codes = slice(0, 16 * d)
    assert np.array_equal(got[..., 16 * d:], want[..., 16 * d:])
    for shift in (0, 4):
        a, b = got[..., codes] >> shift & 15, want[..., codes] >> shift & 15
        assert np.array_equal(np.where(a == 8, 0, a), np.where(b == 8, 0, b))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,d,size", [(8, 128, 64), (1, 64, 16), (3, 128, 48), (5, 64, 256)])
@pytest.mark.parametrize("tokens", [1, 3, 17, 130])
def test_write_and_read(gpu, dtype, heads, d, size, tokens):
    g = torch.Generator().manual_seed(tokens)
    n_pages = -(-200 // size) + 1
    fused = torch.stack([_rows(tokens, heads, d, dtype, 2 * tokens + i) for i in range(2)], 1)
    slots = torch.randperm(n_pages * size, generator=g)[:tokens]
    slots[::5] = torch.tensor([-1, n_pages * size, 2**40, -(2**40)])[torch.arange(len(slots[::5])) % 4]
    before = torch.randint(0, 256, (n_pages, heads, size // 16, 17 * d), generator=g).to(torch.uint8)
    want = _written(before.numpy().copy(), slots.tolist(), fused[:, 0], fused[:, 1], size)
    cache, on_gpu, slots_gpu = before.to(gpu), fused.to(gpu), slots.to(gpu)
    quantized_cache_write(on_gpu[:, 0], on_gpu[:, 1], slots_gpu, cache)
    got = cache.cpu().numpy()
    _same_bytes(got, want, d)
    k, v = quantized_cache_read(cache, slots_gpu, dtype)
    there = (slots >= 0) & (slots < n_pages * size)
    for x, y in ((k, fused[:, 0]), (v, fused[:, 1])):
        assert x.dtype is dtype and torch.equal(x.cpu().double()[there], values(*quantize(y))[there]) and (x.cpu()[~there] == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 64), (F16, 128)])
@pytest.mark.parametrize("first", [0, 3, 16, 29])
def test_neighbours_and_other_orders(gpu, dtype, d, first):
    """Runs of neighbouring slots that begin and end inside of 16, two requests' end to end, and the same backwards."""
    heads, size, n = 4, 32, 90
    x = [_rows(n, heads, d, dtype, i) for i in range(2)]
    slots = torch.cat([torch.arange(first, first + 50), torch.arange(200, 200 + n - 50)])
    for order in (slice(None), torch.arange(n - 1, -1, -1), torch.randperm(n, generator=torch.Generator().manual_seed(1))):
        cache = torch.zeros(10, heads, size // 16, 17 * d, dtype=torch.uint8, device=gpu)
        at = slots[order]
        k, v = (t[order].contiguous() for t in x)
        quantized_cache_write(k.to(gpu), v.to(gpu), at.to(gpu), cache)
        _same_bytes(cache.cpu().numpy(), _written(np.zeros(tuple(cache.shape), dtype=np.uint8), at.tolist(), k, v, size), d)
        got = quantized_cache_read(cache, at.to(gpu), dtype)
        assert all(torch.equal(a.cpu().double(), values(*quantize(b))) for a, b in zip(got, (k, v)))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_types_ends(gpu, dtype):
    """The largest and smallest numbers, and blocks that are no number: their neighbours in the row are what they were."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = _rows(12, 2, 64, dtype, 3)
    rows[0] = big
    rows[1, :, ::2] = -big
    rows[2] = torch.linspace(-1, 1, 64).to(dtype) * big
    rows[3] = tiny
    rows[4] = torch.randint(-9, 10, (64,), generator=torch.Generator().manual_seed(0)).to(dtype) * (tiny * 2.0**-7)  # not normal
    rows[5, 0, 3] = float("inf")
    rows[6, 1, 40] = float("nan")
    rows[7, 0, 63], rows[7, 0, 62] = float("-inf"), big
    cache, slots = quantized_cache_pages(3, 16, 2, 64, gpu), torch.arange(20, 32, device=gpu)
    quantized_cache_write(rows.to(gpu), rows.flip(0).contiguous().to(gpu), slots, cache)
    for got, x in zip(quantized_cache_read(cache, slots, dtype), (rows, rows.flip(0))):
        want = values(*quantize(x))
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().double().nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))
        assert int(torch.isnan(want).sum()) == 3 * 32


def test_read_in_the_other_type(gpu):
    """What bf16 wrote and fp16 does not hold is rounded to it, to infinity past its end."""
    x = _rows(40, 2, 128, BF16, 7)
    x[0], x[1], x[2] = 1e30, 2.0**-30, 3 * 2.0**-26
    cache, slots = quantized_cache_pages(3, 16, 2, 128, gpu), torch.arange(40, device=gpu)
    quantized_cache_write(x.to(gpu), x.to(gpu), slots, cache)
    for got in quantized_cache_read(cache, slots, F16):
        assert torch.equal(got.cpu(), values(*quantize(x)).to(F16))


def test_strides_and_out(gpu):
    heads, d, size, n = 3, 128, 32, 50
    wide = torch.full((7, heads + 1, size // 16, 17 * d), 9, dtype=torch.uint8, device=gpu)
    cache = wide[1:, 1:]
    fused = torch.randn(n, 4 * heads, d + 8, device=gpu).to(F16)
    k, v = fused[:, heads : 2 * heads, :d], fused[:, 2 * heads : 3 * heads, :d]
    slots = torch.randperm(6 * size, device=gpu)[:n]
    quantized_cache_write(k, v, slots, cache)
    want = quantized_cache_pages(6, size, heads, d, gpu).fill_(9)
    quantized_cache_write(k.contiguous(), v.contiguous(), slots, want)
    assert torch.equal(cache, want) and (wide[0] == 9).all() and (wide[:, 0] == 9).all()
    store = torch.full((n, 2, heads, d + 8), 5.0, dtype=F16, device=gpu)
    out = store[:, 0, :, :d], store[:, 1, :, :d]
    got = quantized_cache_read(cache, slots, out=out)
    assert got[0] is out[0] and all(torch.equal(a, b) for a, b in zip(got, quantized_cache_read(want, slots, F16))) and (store[..., d:] == 5).all()


def test_past_32_bits(gpu):
    n_pages, size, heads, d = 70_000, 64, 8, 128  # 4.9 GB
    cache = torch.empty(n_pages, heads, size // 16, 17 * d, dtype=torch.uint8, device=gpu)
    assert cache.numel() > 2**32
    x = [_rows(3, heads, d, BF16, i) for i in range(2)]
    slots = torch.tensor([(n_pages - 1) * size + 63, 30_000 * size, 59_000 * size + 17])
    quantized_cache_write(x[0].to(gpu), x[1].to(gpu), slots.to(gpu), cache)
    got = quantized_cache_read(cache, slots.to(gpu))
    assert all(torch.equal(a.cpu().double(), values(*quantize(b))) for a, b in zip(got, x))


def test_nothing(gpu):
    cache = quantized_cache_pages(2, 16, 2, 64, gpu)
    none, slots = torch.empty(0, 2, 64, dtype=BF16, device=gpu), torch.empty(0, dtype=torch.int64, device=gpu)
    quantized_cache_write(none, none, slots, cache)
    assert [tuple(x.shape) for x in quantized_cache_read(cache, slots)] == [(0, 2, 64)] * 2
    some = torch.ones(3, 2, 64, dtype=BF16, device=gpu)
    quantized_cache_write(some, some, torch.zeros(3, dtype=torch.int64, device=gpu) - 1, cache[:0])
    assert all((x == 0).all() for x in quantized_cache_read(cache[:0], torch.zeros(3, dtype=torch.int64, device=gpu)))
    assert (cache == 0).all()


def test_refusals(gpu):
    cache = quantized_cache_pages(4, 16, 2, 64, gpu)
    k, slots = torch.zeros(3, 2, 64, dtype=BF16, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    good = dict(k=k, v=k, slot_mapping=slots, cache=cache)
    for wrong in (dict(k=k.half()), dict(k=k[:2]), dict(v=k[:, :1]), dict(slot_mapping=slots.int()), dict(slot_mapping=slots[:2]), dict(cache=cache.int()),
                  dict(cache=cache[0]), dict(cache=cache[..., :-1]), dict(cache=cache.transpose(2, 3)), dict(k=k.cpu()), dict(cache=cache.cpu()),
                  dict(k=k.float(), v=k.float()), dict(k=k.transpose(1, 2), v=k.transpose(1, 2)), dict(cache=quantized_cache_pages(4, 16, 2, 128, gpu)),
                  dict(cache=quantized_cache_pages(4, 16, 3, 64, gpu)), dict(k=k.flatten()[4:].new_zeros(4 + 384)[4:].view(3, 2, 64), v=k), dict(k=None)):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            quantized_cache_write(**{**good, **wrong})
    for wrong in (dict(slot_mapping=slots.int()), dict(slot_mapping=slots.view(3, 1)), dict(cache=cache.cpu()), dict(dtype=torch.float32), dict(out=(k, k[:2])),
                  dict(out=(k.float(), k.float())), dict(slot_mapping=slots.cpu())):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            quantized_cache_read(**{**dict(cache=cache, slot_mapping=slots), **wrong})
    for wrong in ((4, 24, 2, 64), (4, 0, 2, 64), (4, 16, 2, 96)):
        with pytest.raises(ValueError):
            quantized_cache_pages(*wrong, gpu)


@pytest.mark.parametrize("window,n_starting", [(None, 0), (20, 3)])
def test_steps_of_answering(gpu, window, n_starting):
    """Prompts and then token after token through tables, writes and attention, against attention over what was kept; requests
    that rest and padding among them."""
    g = torch.Generator().manual_seed(1)
    heads, kv_heads, d, size, batch = 4, 2, 64, 16, 4
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cache = quantized_cache_pages(64, size, kv_heads, d, gpu).fill_(0xFF)
    table = torch.full((batch, 12), -1, dtype=torch.int32, device=gpu)
    free = torch.randperm(64, generator=g).int().to(gpu)
    lens, kept = i32([0] * batch), [[] for _ in range(batch)]
    for new in ([30, 1, 0, 0], [1, 1, 17, 0], [1, 1, 1, 0], [1, 0, 1, 0], [5, 2, 40, 0], [1, 1, 1, 0]):
        n = sum(new) + 3  # padded
        qkv = torch.randn(n, heads + 2 * kv_heads, d, generator=g).to(BF16).to(gpu)
        q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
        made = paged_cache_tables(lens, i32(new), table, free, size, n)
        quantized_cache_write(k, v, made.slot_mapping, cache)
        held = [x.double() for x in quantized_cache_read(cache, made.slot_mapping)]
        assert all(torch.equal(a[: sum(new)].cpu(), values(*quantize(b.cpu()))[: sum(new)]) for a, b in zip(held, (k, v)))
        out, _ = quantized_cache_attention(q, cache, table, made.seq_lens, cu_seqlens_q=made.cu_seqlens, max_seqlen_q=max(new), window=window,
                                           n_starting=n_starting)
        lens, free = made.seq_lens, free[made.pages_taken.item():]
        at = 0
        for b, count in enumerate(new):
            kept[b] += [(held[0][at + i], held[1][at + i]) for i in range(count)]
            for i in range(count):
                x = len(kept[b]) - count + i
                see = [j for j in range(x + 1) if window is None or j < n_starting or j > x - window]
                for h in range(heads):
                    s = torch.stack([kept[b][j][0][h // 2] for j in see]) @ q[at + i, h].double() * d**-0.5
                    rows = torch.stack([kept[b][j][1][h // 2] for j in see])
                    p = torch.softmax(s, 0)
                    # weights and result rounded by half a step each; sums of at most 64 + 97 terms in 32 bits
                    tol = 2.0**-8 * 1.01 * (p @ rows.abs() + (p @ rows).abs()) + 2.0**-12
                    assert ((out[at + i, h].double() - p @ rows).abs() <= tol).all(), (new, b, i, h)
            at += count
    assert table[3].tolist() == [-1] * 12


def test_a_captured_step(gpu):
    """Tables, write, read and attention in one graph whose replays go on from each other's state."""
    size, batch, heads, d = 16, 3, 2, 64
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cache = quantized_cache_pages(40, size, heads, d, gpu)
    lens, new, table = i32([30, 0, 15]), i32([1, 1, 1]), torch.full((batch, 5), -1, dtype=torch.int32, device=gpu)
    table[0, :2], table[2, 0] = i32([7, 3]), 9
    free = i32([20, 21, 22, 23, 24, 25])
    qkv = torch.zeros(batch, 3, heads, d, dtype=F16, device=gpu)

    def step():
        made = paged_cache_tables(lens, new, table, free, size, batch)
        quantized_cache_write(qkv[:, 1], qkv[:, 2], made.slot_mapping, cache)
        return made, quantized_cache_read(cache, made.slot_mapping, F16), quantized_cache_attention(qkv[:, 0], cache, table, made.seq_lens)

    start = cache.clone(), table.clone()
    step()
    cache.copy_(start[0]), table.copy_(start[1])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        made, kv, (out, lse) = step()
    for turn in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(turn)))
        saved = [t.clone() for t in (cache, table)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (cache, table, made.slot_mapping, *kv, out, lse)]
        cache.copy_(saved[0]), table.copy_(saved[1])
        eager, eager_kv, (eager_out, eager_lse) = step()
        for a, b in zip(got, (cache, table, eager.slot_mapping, *eager_kv, eager_out, eager_lse)):
            assert torch.equal(a, b)
        lens.copy_(eager.seq_lens)
        free.copy_(torch.cat([free[eager.pages_taken.item():], free.new_full((eager.pages_taken.item(),), 39)]))
