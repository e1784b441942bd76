"""The tables of a paged cache, the writes through them, and whole steps of answering on the GPU."""

import numpy as np
import pytest
import torch

from dcp_amd.flash_attn_interface import paged_cache_attention
from dcp_amd.ops import paged_cache_tables, paged_cache_write
from tests.paged_cases import tables_truth

pytestmark = pytest.mark.gpu


def _i32(x, gpu):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=gpu)


def _tables(gpu, cached, new, page_size, width, n_free, pad=0, seed=0):
    rng = np.random.default_rng(seed)
    pages = rng.permutation(len(cached) * width + n_free + 1).astype(np.int32)
    table = np.full((len(cached), width), -7, dtype=np.int32)
    for b, c in enumerate(cached):
        have = min(-(-max(c, 0) // page_size), width)
        table[b, :have], pages = pages[:have], pages[have:]
    free = pages[:n_free]
    n_tokens = max(0, int(np.maximum(new, 0).sum()) + pad)
    want, want_table = tables_truth(cached, new, table, free, page_size, n_tokens)
    on_gpu = _i32(table, gpu)
    got = paged_cache_tables(_i32(cached, gpu), _i32(new, gpu), on_gpu, _i32(free, gpu), page_size, n_tokens)
    for name, values in want.items():
        assert getattr(got, name).tolist() == values, name
    assert np.array_equal(on_gpu.cpu().numpy(), want_table)


@pytest.mark.parametrize("cached,new,page_size,width,n_free,pad", [
    ([0], [1], 16, 1, 1, 0),
    ([15, 16, 17, 31, 0], [1, 1, 1, 1, 1], 16, 4, 9, 0),
    ([5, 0, 100, 7], [0, 0, 0, 0], 16, 8, 3, 2),  # nobody adds anything
    ([3, 0, 64, 10, 0], [200, 0, 65, 1, 33], 64, 6, 20, 5),
    ([3, 0, 64, 10, 0], [200, 0, 65, 1, 33], 1, 210, 400, 0),
    ([3, 0, 50], [200, 9, 65], 48, 6, 4, 0),  # too few free pages
    ([3, 0, 50], [200, 9, 65], 16, 6, 0, 0),  # none
    ([90, 0], [200, 300], 64, 3, 9, 1),  # past the rows' width
    ([500, 0], [4, 4], 64, 3, 9, 0),  # cached past it already
    ([-5, 7, -1], [3, -2, -9], 16, 2, 5, 1),
    ([3, 0, 64, 10, 0], [200, 0, 65, 1, 33], 64, 6, 20, -50),  # tokens that do not fit
    ([], [], 64, 3, 2, 3),
    (list(range(0, 2600, 2)), [i % 3 for i in range(1300)], 16, 180, 1000, 7),  # several requests a thread
    ([i % 40 for i in range(257)], [1] * 257, 16, 4, 200, 0),
    ([0] * 256, [900 + i % 7 for i in range(256)], 64, 16, 5000, 100),
])
def test_tables(gpu, cached, new, page_size, width, n_free, pad):
    _tables(gpu, cached, new, page_size, width, n_free, pad)


def test_tables_of_random_lengths(gpu):
    rng = np.random.default_rng(5)
    for seed in range(12):
        n = int(rng.integers(1, 700))
        cached, new = rng.integers(0, 400, n).tolist(), (rng.integers(0, 90, n) * rng.integers(0, 2, n)).tolist()
        _tables(gpu, cached, new, int(rng.choice([1, 16, 48, 64])), int(rng.integers(1, 40)), int(rng.integers(0, 3000)), int(rng.integers(0, 9)), seed)


def test_tables_of_thousands_of_requests(gpu):
    rng = np.random.default_rng(3)
    for n in (1024, 1025, 3001):
        _tables(gpu, rng.integers(0, 100, n).tolist(), rng.integers(0, 3, n).tolist(), 16, 9, 2000, 5, n)


def test_tables_with_lengths_near_the_types_end(gpu):
    """Sums that pass 32 bits: no token is entered twice, nothing outside of the tables is touched."""
    most = 2**31 - 1
    table = torch.full((3, 5), -1, dtype=torch.int32, device=gpu)
    got = paged_cache_tables(_i32([most, 0, most], gpu), _i32([most, most, 4], gpu), table, _i32(range(9), gpu), 16, 100)
    # (the first request's tokens come first, past the width of its row)
    assert got.slot_mapping.tolist() == [-1] * 100 and got.cu_seqlens.tolist() == [0, most, most, most]
    assert got.seq_lens.tolist() == [most, most, most] and got.pages_taken.tolist() == [5]
    assert table.tolist() == [[-1] * 5, [0, 1, 2, 3, 4], [-1] * 5]


def test_tables_take_strided_rows_and_out(gpu):
    wide = torch.full((3, 9), -3, dtype=torch.int32, device=gpu)
    cached, new, free = _i32([0, 0, 0], gpu), _i32([20, 1, 40], gpu), _i32([5, 4, 3, 2, 1, 0], gpu)
    first = paged_cache_tables(cached, new, wide[:, 2:5], free, 16, 61)
    assert wide[:, 2:5].tolist() == [[5, 4, -3], [3, -3, -3], [2, 1, 0]] and (wide[:, :2] == -3).all() and (wide[:, 5:] == -3).all()
    again = paged_cache_tables(cached, new, wide[:, 2:5], free, 16, 61, out=first)
    assert again.slot_mapping.data_ptr() == first.slot_mapping.data_ptr() and again.pages_taken.tolist() == [6]
    for wrong in (dict(block_table=wide[:, :3].t()), dict(block_table=wide[:1, :3].expand(3, 3)), dict(block_table=wide[:, :3].long()),
                  dict(new_lens=new[:2]), dict(cached_lens=cached.cpu()), dict(page_size=0), dict(n_tokens=-1), dict(n_tokens=60, out=first),
                  dict(cached_lens=first.seq_lens, out=first), dict(free_pages=free.view(2, 3))):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            paged_cache_tables(**{**dict(cached_lens=cached, new_lens=new, block_table=wide[:, 2:5], free_pages=free, page_size=16, n_tokens=61), **wrong})


@pytest.mark.parametrize("dtype,heads,head_dim", [(torch.bfloat16, 8, 128), (torch.float16, 1, 64), (torch.float32, 3, 40), (torch.bfloat16, 5, 7),
                                                  (torch.uint8, 2, 33), (torch.bfloat16, 2, 6)])
@pytest.mark.parametrize("tokens", [1, 3, 4, 130])
def test_write(gpu, dtype, heads, head_dim, tokens):
    g = torch.Generator().manual_seed(tokens)
    n_pages, size = 12, 16
    make = lambda *shape: torch.randint(0, 200, shape, generator=g).to(dtype)
    fused, store = make(tokens, 2, heads, head_dim), make(n_pages, size, 2, heads, head_dim)
    slots = torch.randperm(n_pages * size, generator=g)[:tokens]
    slots[::5] = torch.tensor([-1, n_pages * size, 2**40, -(2**40)])[torch.arange(len(slots[::5])) % 4]
    want = store.clone()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < n_pages * size:
            want[slot // size, slot % size] = fused[t]
    fused, on_gpu, slots = fused.to(gpu), store.to(gpu), slots.to(gpu)
    paged_cache_write(fused[:, 0], fused[:, 1], slots, on_gpu[:, :, 0], on_gpu[:, :, 1])
    assert torch.equal(on_gpu.cpu(), want)
    apart = store.permute(2, 0, 3, 1, 4).contiguous().to(gpu)  # heads before a page's tokens
    paged_cache_write(fused[:, 0].clone(), fused[:, 1].clone(), slots, apart[0].transpose(1, 2), apart[1].transpose(1, 2))
    assert torch.equal(apart.cpu(), want.permute(2, 0, 3, 1, 4))


def test_write_past_32_bits(gpu):
    cache = torch.empty(80_000, 64, 2, 2, 128, dtype=torch.bfloat16, device=gpu)
    k, v = (torch.randn(2, 2, 128, device=gpu).to(torch.bfloat16) for _ in range(2))
    slots = [79_999 * 64 + 63, 40_000 * 64]
    paged_cache_write(k, v, torch.tensor(slots, device=gpu), cache[:, :, 0], cache[:, :, 1])
    assert torch.equal(cache[79_999, 63, 0], k[0]) and torch.equal(cache[79_999, 63, 1], v[0])
    assert torch.equal(cache[40_000, 0, 0], k[1]) and torch.equal(cache[40_000, 0, 1], v[1])


def test_write_refusals(gpu):
    cache = torch.zeros(4, 16, 2, 2, 64, dtype=torch.bfloat16, device=gpu)
    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    good = dict(k=k, v=k, slot_mapping=slots, k_cache=cache[:, :, 0], v_cache=cache[:, :, 1])
    for wrong in (dict(k=k.half()), dict(k=k[:2]), dict(v=k[:, :1]), dict(slot_mapping=slots.int()), dict(slot_mapping=slots[:2]),
                  dict(v_cache=cache[:, :, 1].contiguous()), dict(k_cache=cache), dict(k=k.cpu()), dict(k=k.transpose(1, 2), v=k.transpose(1, 2))):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            paged_cache_write(**{**good, **wrong})
    with pytest.raises(AssertionError, match="element size"):
        paged_cache_write(k.double(), k.double(), slots, cache[:, :, 0].double(), cache[:, :, 1].double())


@pytest.mark.parametrize("window,n_starting", [(None, 0), (20, 3)])
def test_steps_of_answering(gpu, window, n_starting):
    """Prompts and then token after token through tables, writes and attention, against attention over the kept keys; requests
    that rest and a last, padding one among them."""
    g = torch.Generator().manual_seed(1)
    heads, kv_heads, d, size, batch = 4, 2, 64, 16, 4
    cache = torch.full((64, size, 2, kv_heads, d), float("nan"), dtype=torch.bfloat16, device=gpu)
    table = torch.full((batch, 12), -1, dtype=torch.int32, device=gpu)
    free = torch.randperm(64, generator=g).int().to(gpu)
    lens, kept = _i32([0] * batch, gpu), [[] for _ in range(batch)]
    for new in ([30, 1, 0, 0], [1, 1, 17, 0], [1, 1, 1, 0], [1, 0, 1, 0], [5, 2, 40, 0], [1, 1, 1, 0]):
        n = sum(new) + 3  # padded
        qkv = torch.randn(n, heads + 2 * kv_heads, d, generator=g).to(torch.bfloat16).to(gpu)
        q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
        made = paged_cache_tables(lens, _i32(new, gpu), table, free, size, n)
        paged_cache_write(k, v, made.slot_mapping, cache[:, :, 0], cache[:, :, 1])
        out, _ = paged_cache_attention(q, cache[:, :, 0], cache[:, :, 1], table, made.seq_lens, cu_seqlens_q=made.cu_seqlens,
                                       max_seqlen_q=max(new), window=window, n_starting=n_starting)
        lens, free = made.seq_lens, free[made.pages_taken.item():]
        at = 0
        for b, count in enumerate(new):
            kept[b] += [(k[at + i].double(), v[at + i].double()) for i in range(count)]
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
    """Tables, write and attention in one graph whose replays go on from each other's state."""
    size, batch, heads, d = 16, 3, 2, 64
    cache = torch.zeros(40, size, 2, heads, d, dtype=torch.float16, device=gpu)
    lens, new, table = _i32([30, 0, 15], gpu), _i32([1, 1, 1], gpu), torch.full((batch, 5), -1, dtype=torch.int32, device=gpu)
    table[0, :2], table[2, 0] = _i32([7, 3], gpu), 9
    free = _i32([20, 21, 22, 23, 24, 25], gpu)
    qkv = torch.zeros(batch, 3, heads, d, dtype=torch.float16, device=gpu)

    def step():
        made = paged_cache_tables(lens, new, table, free, size, batch)
        paged_cache_write(qkv[:, 1], qkv[:, 2], made.slot_mapping, cache[:, :, 0], cache[:, :, 1])
        return made, paged_cache_attention(qkv[:, 0], cache[:, :, 0], cache[:, :, 1], table, made.seq_lens)

    start = cache.clone(), table.clone()
    step()
    cache.copy_(start[0]), table.copy_(start[1])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        made, (out, lse) = step()
    for turn in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(turn)))
        saved = [t.clone() for t in (cache, table)]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (cache, table, made.slot_mapping, out, lse)]
        cache.copy_(saved[0]), table.copy_(saved[1])
        eager, (eager_out, eager_lse) = step()
        for a, b in zip(got, (cache, table, eager.slot_mapping, eager_out, eager_lse)):
            assert torch.equal(a, b)
        lens.copy_(eager.seq_lens)
        free.copy_(torch.cat([free[eager.pages_taken.item():], free.new_full((eager.pages_taken.item(),), 39)]))
