"""Attention over a paged cache held in 4 bits on the GPU, against its definition in 64 bits.  Bytes of every place of the cache that no
query of its request sees are 0xff: no numbers."""

import math

import pytest
import torch

from dcp_amd.flash_attn_interface import paged_cache_attention, quantized_cache_attention, quantized_cache_workspace_bytes
from dcp_amd.ops import quantized_cache_pages, quantized_cache_read, quantized_cache_write
from tests.paged_cases import check
from tests.quantized_cases import Quantized
from tests.test_paged_attention_gpu import SINGLE, TOKENS, WINDOWS

pytestmark = pytest.mark.gpu
F16 = torch.float16
CASES = {**SINGLE, **WINDOWS, **TOKENS}


def _run(gpu, case, sentinel=None, **more):
    args = {**case.to(gpu), **more}
    if sentinel is not None:
        args.update(out=torch.full_like(args["q"], sentinel), lse=torch.full(args["q"].shape[1::-1], sentinel, device=gpu))
    got = quantized_cache_attention(**args)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("name", CASES)
def test_against_64_bits(gpu, name):
    case = Quantized(**CASES[name])
    check(_run(gpu, case), case.truth())


@pytest.mark.parametrize("longest", [1, 64, 700, 5000, 1 << 20])
@pytest.mark.parametrize("name", ["short", "empty_rows", "long", "long_window", "chunk", "mixed", "group_24", "fp16_d64", "window_and_first", "few"])
def test_lengths_the_host_does_not_know(gpu, name, longest):
    """max_seqlen_k splits the work and no more, too short or too long."""
    case = Quantized(**CASES[name])
    check(_run(gpu, case, max_seqlen_k=longest), case.truth())


@pytest.mark.parametrize("longest_q", [1, 5, 1000])
@pytest.mark.parametrize("name", ["few", "five_heads", "mixed", "chunk", "window_chunk", "more_tokens_than_keys", "many"])
def test_numbers_of_tokens_the_host_does_not_know(gpu, name, longest_q):
    """max_seqlen_q chooses a kernel and no more."""
    case = Quantized(**CASES[name])
    args = case.to(gpu)
    if "cu_seqlens_q" not in args:
        args["cu_seqlens_q"] = torch.tensor(case.cu, dtype=torch.int32, device=gpu)
    check(quantized_cache_attention(**{**args, "max_seqlen_q": longest_q}), case.truth())


@pytest.mark.parametrize("requests", [63, 64, 65, 130])
def test_row_tiles_of_many_requests(gpu, requests):
    """Requests without tokens, with a part of a tile of rows and with several."""
    new = [(0, 3, 17, 64, 65)[(i * 7 + i // 5) % 5] for i in range(requests)]
    case = Quantized([n + (i * 13) % 60 for i, n in enumerate(new)], new=new, heads=4, kv_heads=2, head_dim=64, page_size=16)
    check(_run(gpu, case), case.truth())


RAGGED = {
    "ragged": dict(keys=[3000, 17, 900, 0, 64, 5, 1500], new=[40, 17, 0, 0, 30, 9, 33]),
    "five_kv_heads": dict(keys=[2100, 700, 90], new=[30, 60, 90], heads=25, kv_heads=5, head_dim=64),
    "window": dict(keys=[2500, 100, 1300], new=[70, 100, 200], heads=4, kv_heads=2, window=300, n_starting=70),
    "fp16": dict(keys=[1800, 250], new=[300, 9], heads=4, kv_heads=4, dtype=F16),
    "rows_of_many_heads": dict(keys=[1400, 300, 20], new=[9, 300, 3], heads=48, kv_heads=1, head_dim=64),
    "more_tokens_than_keys": dict(keys=[10, 1100, 0], new=[150, 40, 60], heads=4, kv_heads=2),
    "alone": dict(keys=[5000], new=[50], heads=8, kv_heads=1, page_size=16),
    "at_most_64_rows": dict(keys=[3000, 17, 900, 0, 64, 1500], new=[16, 9, 0, 3, 16, 1]),
    "at_most_64_rows_fp16_d64": dict(keys=[2500, 40, 1300], new=[13, 13, 12], heads=25, kv_heads=5, head_dim=64, dtype=F16),
    "at_most_64_rows_window": dict(keys=[2500, 100, 1300], new=[33, 30, 64], heads=3, kv_heads=3, head_dim=64, window=300, n_starting=70),
}


@pytest.mark.parametrize("longest", [1, 200, 1 << 20])
@pytest.mark.parametrize("name", RAGGED)
def test_ragged_prompts(gpu, name, longest):
    """Row tiles taken whole, those that see the most first, and cut into pieces of about one length."""
    case = Quantized(**RAGGED[name])
    args = case.to(gpu)
    wide = torch.full((len(case.keys), 3000), -1, dtype=torch.int32, device=gpu)  # (and of tables with more room than there are keys)
    wide[:, : args["block_table"].shape[1]] = args["block_table"]
    truth = case.truth()
    for table in (args["block_table"], wide):
        check(_run(gpu, case, sentinel=5.0, max_seqlen_k=longest, block_table=table), truth)


@pytest.mark.parametrize("longest_q", [9, 16, 100])
@pytest.mark.parametrize("requests", [5, 70])
def test_tiles_of_rows_the_host_does_not_know(gpu, requests, longest_q):
    """36 rows are taken by tiles of 64, 400 by tiles of 128, whatever the requests have."""
    new = [(0, 3, 17, 40, 9)[i % 5] for i in range(requests)]
    case = Quantized([n + (i * 37) % 200 for i, n in enumerate(new)], new=new, heads=4, kv_heads=1, head_dim=64, page_size=16)
    for longest in (64, 100000):
        check(_run(gpu, case, max_seqlen_q=longest_q, max_seqlen_k=longest), case.truth())


@pytest.mark.parametrize("new", [[1] * 64, [33] * 64, [0] * 63 + [200]])
def test_pieces_of_as_many_requests_as_a_wave_looks_at(gpu, new):
    case = Quantized([n + (i * 37) % 200 for i, n in enumerate(new)], new=new, heads=2, kv_heads=1, head_dim=64, page_size=16)
    check(_run(gpu, case, max_seqlen_q=max(max(new), 33), max_seqlen_k=100000), case.truth())


def test_a_batch_of_thousands(gpu):
    """Requests past the 64 that a wave looks at together, some of no tokens and no keys among them."""
    n = 1500
    case = Quantized([(i * 7) % 40 for i in range(n)], new=[i % 3 for i in range(n)], heads=2, kv_heads=1, head_dim=64, page_size=16)
    truth = case.truth()
    for longest_q in (1, 2, 100):
        for longest_k in (48, 5000):
            check(_run(gpu, case, max_seqlen_q=longest_q, max_seqlen_k=longest_k), truth)


@pytest.mark.parametrize("keys", [64, 65])
def test_shares_that_end_with_a_request(gpu, keys):
    """Many requests of the same length: few are cut, or nearly all are."""
    case = Quantized([keys] * 1024, heads=2, kv_heads=1, head_dim=64, page_size=16)
    check(_run(gpu, case, max_seqlen_k=5000), case.truth())


@pytest.mark.parametrize("requests", [65536, 65600])
def test_tens_of_thousands_of_requests(gpu, requests):
    n, n_pages = requests, 4
    x = torch.randn(2, n_pages * 16, 1, 64, device=gpu).to(torch.bfloat16)
    cache, slots = quantized_cache_pages(n_pages, 16, 1, 64, gpu), torch.arange(n_pages * 16, device=gpu)
    quantized_cache_write(x[0], x[1], slots, cache)
    k, v = (t.view(n_pages, 16, 64).double() for t in quantized_cache_read(cache, slots))
    q = torch.randn(n, 1, 64, device=gpu).to(torch.bfloat16)
    table = torch.arange(n, dtype=torch.int32, device=gpu)[:, None] % n_pages
    lens = torch.arange(n, dtype=torch.int32, device=gpu) % 17
    got = quantized_cache_attention(q, cache, table, lens)
    k64, v64 = (t[table[:, 0].long()] for t in (k, v))
    s = (q.double() * k64).sum(-1) * 64**-0.5
    s.masked_fill_(torch.arange(16, device=gpu) >= lens[:, None], -math.inf)
    weights = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e30))
    total = weights.sum(1)
    truth = ((weights[..., None] * v64).sum(1) / total.clamp_min(1e-300)[:, None])[:, None]
    # weights and results are rounded to bf16, half a step each, of values up to the largest |v| (and fp32 sums of 80 terms)
    assert (got[0].double() - truth).abs().max() <= (2 * 2.0**-8 + 2.0**-15) * v64.abs().max()
    some = lens > 0
    lse = s.amax(1) + total.log()
    assert (got[1][0][some].double() - lse[some]).abs().max() <= 2.0**-16 * (1 + lse[some].abs().max())
    assert torch.isinf(got[1][0][~some]).all() and (got[0][~some] == 0).all()


@pytest.mark.parametrize("new", [None, [3, 200]])
def test_strides(gpu, new):
    case = Quantized([70, 300], new=new, page_size=32)
    args = case.to(gpu)
    q = torch.empty(len(case.q), case.heads + 4, case.head_dim + 8, dtype=case.dtype, device=gpu)[:, 2:-2, 8:]
    q.copy_(args["q"])
    table = torch.full((2, args["block_table"].shape[1] + 3), -1, dtype=torch.int32, device=gpu)[:, 1:-2]
    table.copy_(args["block_table"])
    cache = torch.full((case.n_pages + 2, case.kv_heads + 3, 2, 17 * case.head_dim), 0xFF, dtype=torch.uint8, device=gpu)[1:-1, 2:-1]
    cache.copy_(args["cache"])
    store = torch.full((len(case.q), case.heads, 2 * case.head_dim), 7.0, dtype=case.dtype, device=gpu)
    args.update(q=q, block_table=table, cache=cache, out=store[..., : case.head_dim])
    check(quantized_cache_attention(**args), case.truth())
    assert (store[..., case.head_dim:] == 7).all()
    by_head = args["cache"].transpose(0, 1).contiguous().transpose(0, 1)
    check(quantized_cache_attention(**{**args, "cache": by_head}), case.truth())


@pytest.mark.parametrize("kind", ["single", "tokens", "window"])
def test_entries_that_name_no_page(gpu, kind):
    """Their keys are seen by none, wherever in the row they stand."""
    bad = [(0, 1, lambda n: -1), (1, 0, lambda n: n), (1, 3, lambda n: -(2**31)), (2, 0, lambda n: 2**31 - 1)]
    more = dict(single=dict(), tokens=dict(new=[100, 1, 30]), window=dict(window=70, n_starting=3))[kind]
    case = Quantized([300, 333, 30], bad=bad, page_size=32 if kind == "window" else 64, **more)
    check(_run(gpu, case), case.truth())


@pytest.mark.parametrize("longest", [1, 1 << 20])
@pytest.mark.parametrize("window", [0, 9000])
def test_missing_pages_far_into_a_unit(gpu, longest, window):
    """A wave finds its tiles 32 at a time; what is missing of the last of them and of the first of the next."""
    missing = [(0, i, lambda n: -1) for tile in (31 * 4, 31 * 8, 32 * 4 + 3, 63 * 4 + 1, 64 * 8 + 7) for i in (2 * tile,)]
    case = Quantized([17500], bad=missing, page_size=16, heads=2, kv_heads=1, window=window, n_starting=100 if window else 0)
    check(_run(gpu, case, max_seqlen_k=longest), case.truth())


@pytest.mark.parametrize("keys", [[100, 9], [9000, 9]])
@pytest.mark.parametrize("new", [None, [2, 0], [90, 0]])
def test_tokens_of_no_request_are_left(gpu, keys, new):
    case = Quantized(keys, new=new, extra_tokens=5, heads=2, kv_heads=1)
    check(_run(gpu, case, sentinel=3.0), case.truth(), untouched=3.0)


@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("longest", [64, 100000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, F16])
def test_rounding_of_a_weight_that_outweighs_the_others_cancels(gpu, dtype, longest, group):
    """279 keys of weight 1 and value 0, and behind the first of them one of weight w from 2^12.5 to 2^13.5 and value 1: w / (w + 279).  w is
    rounded by up to eps / 2; were only the product's w, the result would be off by that.  Where the sum's is as well, 279 / (w + 279) < 0.046 of
    it is left, beside half a step of the result (eps / 4 below 1) and sums in 32 bits."""
    batch, kv_heads, d, n = 4, 4, 64, 280
    k, v = (torch.zeros(n, kv_heads, d, dtype=dtype, device=gpu) for _ in range(2))
    k[270, :, 0], k[270, :, 1], v[270] = 6.0, 0.5, 1.0
    cache = quantized_cache_pages(18, 16, kv_heads, d, gpu)
    quantized_cache_write(k, v, torch.arange(n, device=gpu), cache)
    g = torch.Generator().manual_seed(1)
    q = torch.zeros(batch, kv_heads * group, d)
    q[..., 0], q[..., 1] = 11.5625, torch.rand(q.shape[:2], generator=g) * 10
    q = q.to(dtype)
    table, lens = torch.arange(18, dtype=torch.int32, device=gpu).expand(batch, 18).contiguous(), torch.full((batch,), n, dtype=torch.int32, device=gpu)
    cu = torch.arange(batch + 1, dtype=torch.int32, device=gpu)
    out, lse = quantized_cache_attention(q.to(gpu), cache, table, lens, cu_seqlens_q=cu, max_seqlen_q=1, max_seqlen_k=longest)
    w = torch.exp((6 * q[..., 0].double() + 0.5 * q[..., 1].double()) * d**-0.5)
    assert w.log2().min() > 12.5 and w.log2().max() < 13.5
    off = (out.double().cpu() - (w / (w + n - 1))[..., None]).abs().max()
    eps = torch.finfo(dtype).eps
    assert off <= eps / 4 + 0.046 * eps / 2 + 2.0**-16
    assert (lse.double().cpu().T - (w + n - 1).log()).abs().max() <= 2.0**-18


@pytest.mark.parametrize("before", [4, 300])
@pytest.mark.parametrize("new", [[1, 1], [40, 20]])
def test_tokens_before_the_first_request_are_left(gpu, before, new):
    case = Quantized([90, 40], new=new, heads=2, kv_heads=1)
    args = case.to(gpu)
    q = torch.cat([args["q"].new_zeros(before, 2, 128), args["q"]])
    out, lse = torch.full_like(q, 3.0), torch.full((2, len(q)), 3.0, device=gpu)
    args.update(q=q, cu_seqlens_q=torch.tensor(case.cu + before, dtype=torch.int32, device=gpu), out=out, lse=lse)
    for longest_q in (1, max(new)):
        for longest in (64, 100000):
            quantized_cache_attention(**{**args, "max_seqlen_q": longest_q, "max_seqlen_k": longest})
            assert (out[:before] == 3).all() and (lse[:, :before] == 3).all()
            check((out[before:], lse[:, before:]), case.truth())


def test_no_requests_and_no_pages(gpu):
    args = Quantized([10, 20]).to(gpu)
    none = {**args, "q": args["q"][:0], "block_table": args["block_table"][:0], "seq_lens": args["seq_lens"][:0]}
    out, lse = quantized_cache_attention(**none)
    assert out.shape == (0, 8, 128) and lse.shape == (8, 0)
    for longest_q in (1, 100):
        out, lse = quantized_cache_attention(**{**args, "cache": args["cache"][:0], "max_seqlen_q": longest_q})
        assert (out == 0).all() and (lse == torch.inf).all()


def test_offsets_past_32_bits(gpu):
    """A cache of 5 GB: pages that begin past 2^32 bytes."""
    case = Quantized([500, 77], heads=4, kv_heads=2, page_size=64)
    args, n_pages = case.to(gpu), 300_000
    cache = torch.empty(n_pages, 2, 4, 17 * 128, dtype=torch.uint8, device=gpu)
    last = n_pages - case.n_pages
    cache[last:] = args["cache"]
    args.update(cache=cache, block_table=args["block_table"] + last)
    assert last * cache.stride(0) > 2**32
    check(quantized_cache_attention(**args), case.truth())
    q = torch.randn(80, 4, 128, device=gpu).to(case.dtype)  # (and by the kernel of rows)
    near, far = ({**args, "q": q, "cu_seqlens_q": torch.tensor([0, 70, 80], dtype=torch.int32, device=gpu), "max_seqlen_q": 70, **x}
                 for x in (dict(cache=cache[last:].clone(), block_table=args["block_table"] - last), {}))
    assert all(torch.equal(a, b) for a, b in zip(quantized_cache_attention(**near), quantized_cache_attention(**far)))


@pytest.mark.parametrize("name", ["long", "mixed", "chunk"])
def test_the_same_twice(gpu, name):
    case = Quantized(**CASES[name])
    first, second = _run(gpu, case), _run(gpu, case)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", [torch.bfloat16, F16])
@pytest.mark.parametrize("new", [[1, 1], [70, 20]])
def test_as_over_the_same_cache_in_16_bits(gpu, dtype, new):
    """Read back into a cache of 16 bits, the keys and values give what they give here, up to the order of sums and the weights' rounding."""
    case = Quantized([900, 333], new=new, dtype=dtype)
    args, n = case.to(gpu), case.n_pages * case.page_size
    kv = quantized_cache_read(args["cache"], torch.arange(n, device=gpu), dtype)
    k, v = (x.view(case.n_pages, case.page_size, case.kv_heads, case.head_dim) for x in kv)
    wide = paged_cache_attention(**{name: x for name, x in args.items() if name != "cache"}, k_cache=k, v_cache=v)
    truth = case.truth()
    check(wide, truth)
    check(quantized_cache_attention(**args), truth)


def test_a_block_that_is_no_number_is_seen(gpu):
    """Whoever sees it gets no number; requests that do not are what they were."""
    case = Quantized([300, 200], page_size=16)
    args = case.to(gpu)
    before = quantized_cache_attention(**args)
    cache = args["cache"].clone()
    page, d = int(args["block_table"][0, 3]), case.head_dim
    cache[page, 1, 0, 16 * d + 5 * (d // 32) + 2] = 0xFF  # an exponent of K of head 1
    out, lse = quantized_cache_attention(**{**args, "cache": cache})
    assert torch.isnan(out[0, 4:]).all() and torch.isnan(lse[4:, 0]).all()
    assert torch.equal(out[0, :4], before[0][0, :4]) and torch.equal(out[1], before[0][1]) and torch.equal(lse[:, 1], before[1][:, 1])


@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_a_callers_workspace_is_enough_and_bounded(gpu, new):
    case = Quantized([9000, 20], new=new, heads=2, kv_heads=1)
    args = case.to(gpu)
    n = quantized_cache_workspace_bytes(**args)
    store = torch.full((n + 4096,), 0xEE, dtype=torch.uint8, device=gpu)
    check(quantized_cache_attention(**args, workspace=store[:n]), case.truth())
    assert (store[n:] == 0xEE).all()
    with pytest.raises(AssertionError, match="workspace"):
        quantized_cache_attention(**args, workspace=store[: n - 1])


def test_calls_at_the_same_time(gpu):
    """Two streams, and two graphs with a workspace each, replayed side by side."""
    cases = [Quantized([3000, 9, 700], heads=4, kv_heads=2), Quantized([2500, 130], new=[40, 100], heads=4, kv_heads=2, seed=1)]
    args, truths, streams = [c.to(gpu) for c in cases], [c.truth() for c in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(quantized_cache_attention(**args[i]))
    torch.cuda.synchronize()
    for results, truth in zip(got, truths):
        for result in results:
            check(result, truth)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for i, graph in enumerate(graphs):
        more = dict(out=torch.empty_like(args[i]["q"]), lse=torch.empty(args[i]["q"].shape[1::-1], device=gpu),
                    workspace=torch.empty(max(quantized_cache_workspace_bytes(**args[i]), 1), dtype=torch.uint8, device=gpu))
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=streams[i]):
            quantized_cache_attention(**args[i], **more)
        outs.append(more)
    for _ in range(3):
        for more in outs:
            more["out"].fill_(9)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for more, truth in zip(outs, truths):
            check((more["out"], more["lse"]), truth)


@pytest.mark.parametrize("new", [[1, 1, 1], [60, 1, 40]])
def test_captured_and_replayed_with_other_lengths(gpu, new):
    """One graph for all steps: lengths are read on the device."""
    case = Quantized([2000, 900, 64], new=new, heads=4, kv_heads=2)
    args = case.to(gpu)
    quantized_cache_attention(**args)
    out, lse = torch.empty_like(args["q"]), torch.empty(4, sum(new), device=gpu)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        quantized_cache_attention(**args, out=out, lse=lse)
    for lens in ([2000, 900, 64], [1, 0, 64], [1999, 17, 33], [2000, 900, 64]):
        args["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = quantized_cache_attention(**args)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("wrong", ["q_type", "q_axes", "cache_type", "cache_axes", "cache_dense", "tables", "lens", "cu", "no_cu", "out", "lse", "dim",
                                   "window", "wide_window", "half_a_token", "scale", "huge_scale", "aligned", "cache_aligned", "cpu", "q_cpu", "heads",
                                   "workspace"])
def test_refusals(gpu, wrong):
    case = Quantized([70, 30])
    args = case.to(gpu)
    q, cache, table = args["q"], args["cache"], args["block_table"]
    shifted = torch.zeros(cache.numel() + 8, dtype=torch.uint8, device=gpu)[8:].view(cache.shape)
    change = dict(
        q_type=dict(q=q.float()), q_axes=dict(q=q[0]), cache_type=dict(cache=cache.view(torch.int8)), cache_axes=dict(cache=cache[0]),
        cache_dense=dict(cache=cache[:, :, ::2]), tables=dict(block_table=table.long()), lens=dict(seq_lens=args["seq_lens"][:1]),
        cu=dict(cu_seqlens_q=args["seq_lens"]), no_cu=dict(q=torch.cat([q, q])), out=dict(out=q[:1].clone()), lse=dict(lse=torch.empty(2, 8, device=gpu)),
        dim=dict(q=q[..., :64].contiguous()), window=dict(window=0), wide_window=dict(window=1 << 40), half_a_token=dict(window=9, n_starting=1.5),
        scale=dict(softmax_scale=0.0), huge_scale=dict(softmax_scale=1e39),
        aligned=dict(q=torch.empty(2 * 8 * 128 + 8, dtype=q.dtype, device=gpu)[4 : 4 + 2 * 8 * 128].view(2, 8, 128)), cache_aligned=dict(cache=shifted),
        cpu=dict(cache=cache.cpu()), q_cpu=dict(q=q.cpu()), heads=dict(q=q[:, :5].contiguous()),
        workspace=dict(workspace=torch.empty(16, dtype=torch.uint8, device=gpu), max_seqlen_k=100000))[wrong]
    with pytest.raises((ValueError, TypeError, AssertionError)):
        quantized_cache_attention(**{**args, **change})
