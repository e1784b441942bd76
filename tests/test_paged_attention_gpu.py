"""Attention over a paged cache and over shared prefixes on the GPU, against their definitions in 64 bits.  Every place of the
cache that no query of its request sees holds NaN."""

import math

import pytest
import torch

from dcp_amd.flash_attn_interface import (paged_cache_attention, paged_cache_workspace_bytes, shared_prefix_attention,
                                          shared_prefix_workspace_bytes)
from tests.paged_cases import Paged, check

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _run(gpu, case, sentinel=None, **more):
    args = {**case.to(gpu), **more}
    if sentinel is not None:
        args.update(out=torch.full_like(args["q"], sentinel), lse=torch.full(args["q"].shape[1::-1], sentinel, device=gpu))
    got = (shared_prefix_attention if case.prefixes else paged_cache_attention)(**args)
    torch.cuda.synchronize()
    return got


SINGLE = dict(
    short=dict(keys=[1, 2, 15, 16, 17, 63, 64, 65]),
    empty_rows=dict(keys=[0, 5, 0, 300, 0]),
    one=dict(keys=[1]),
    small_pages=dict(keys=[100, 1, 33, 257, 1000], page_size=16),
    odd_pages=dict(keys=[100, 49, 47, 96, 700], page_size=48),
    long_pages=dict(keys=[1000, 300, 256], page_size=256),
    fp16_d64=dict(keys=[77, 500, 3], head_dim=64, heads=8, kv_heads=8, dtype=F16),
    bf16_d64=dict(keys=[77, 500, 3], head_dim=64, heads=8, kv_heads=2),
    fp16_d128=dict(keys=[77, 500, 3], dtype=F16),
    group_5=dict(keys=[130, 31, 1025], heads=10, kv_heads=2),
    group_16=dict(keys=[130, 31, 1025], heads=16, kv_heads=1),
    group_24=dict(keys=[130, 31, 1025], heads=24, kv_heads=1),
    group_71=dict(keys=[130, 31, 1025], heads=71, kv_heads=1),
    one_head=dict(keys=[130, 31, 1025], heads=1, kv_heads=1),
    many=dict(keys=[(37 * i) % 211 for i in range(300)], heads=2, kv_heads=1, page_size=16),
    long=dict(keys=[9000, 20], heads=2, kv_heads=1),
    longer=dict(keys=[30011], heads=4, kv_heads=2, head_dim=64),
    flat_scores=dict(keys=[500, 40], q_scale=0.0),
    sharp_scores=dict(keys=[500, 40], q_scale=30.0),
)
WINDOWS = dict(
    window_of_one=dict(keys=[1, 2, 17, 64, 300], window=1),
    window=dict(keys=[1, 20, 33, 34, 100, 1000, 64, 0], window=33),
    window_and_first=dict(keys=[1, 5, 37, 38, 39, 54, 100, 1000], window=33, n_starting=5),
    window_at_groups=dict(keys=[256, 257, 512, 48, 79, 80, 81], window=32, n_starting=16, page_size=16),
    first_touch_window=dict(keys=[60, 61, 62, 63, 64, 65, 66, 67], window=40, n_starting=20),
    longer_than_keys=dict(keys=[10, 100], window=5000, n_starting=9000),
    long_window=dict(keys=[5000, 2049, 600], window=1000, n_starting=64, head_dim=64, dtype=F16),
)
TOKENS = dict(
    few=dict(keys=[4, 10, 300], new=[4, 3, 2]),
    five_heads=dict(keys=[8, 300], new=[7, 5], heads=10, kv_heads=2),
    mixed=dict(keys=[10, 1, 5, 200, 300, 64, 0], new=[0, 1, 5, 130, 300, 64, 0]),
    whole_prompts=dict(keys=[257, 33], new=[257, 33], head_dim=64, dtype=F16, heads=4, kv_heads=4),
    more_tokens_than_keys=dict(keys=[3, 0, 20], new=[9, 4, 50]),
    chunk=dict(keys=[1500], new=[300], heads=4, kv_heads=1),
    window_chunk=dict(keys=[700, 150, 90], new=[200, 150, 3], window=50, n_starting=7),
    window_prompt=dict(keys=[400], new=[400], window=17, page_size=16, head_dim=64),
    first_of_long_chunk=dict(keys=[900, 30], new=[260, 30], window=100, n_starting=130, heads=4, kv_heads=2),
)


@pytest.mark.parametrize("name", [*SINGLE, *WINDOWS, *TOKENS])
def test_against_64_bits(gpu, name):
    case = Paged(**{**SINGLE, **WINDOWS, **TOKENS}[name])
    check(_run(gpu, case), case.truth())


@pytest.mark.parametrize("longest", [1, 100, 1 << 20])
@pytest.mark.parametrize("name", ["long", "long_window", "chunk", "mixed"])
def test_lengths_the_host_does_not_know(gpu, name, longest):
    """max_seqlen_k splits the work and no more, too short or too long."""
    case = Paged(**{**SINGLE, **WINDOWS, **TOKENS}[name])
    check(_run(gpu, case, max_seqlen_k=longest), case.truth())


@pytest.mark.parametrize("longest_q", [1, 5, 1000])
@pytest.mark.parametrize("name", ["few", "five_heads", "mixed", "chunk", "window_chunk", "more_tokens_than_keys", "many", "tokens", "no_tokens",
                                  "some_without", "empty_prefix", "no_own_keys"])
def test_numbers_of_tokens_the_host_does_not_know(gpu, name, longest_q):
    """max_seqlen_q chooses a kernel and no more."""
    case = Paged(**{**SINGLE, **WINDOWS, **TOKENS, **PREFIXES}[name])
    args = case.to(gpu)
    if "cu_seqlens_q" not in args:
        args["cu_seqlens_q"] = torch.tensor(case.cu, dtype=torch.int32, device=gpu)
    got = (shared_prefix_attention if case.prefixes else paged_cache_attention)(**{**args, "max_seqlen_q": longest_q})
    check(got, case.truth())


@pytest.mark.parametrize("longest", [64, 700, 5000])
@pytest.mark.parametrize("name", ["short", "empty_rows", "group_24", "fp16_d64", "window_and_first", "first_touch_window", "few", "groups",
                                  "some_without"])
def test_units_whole_and_cut(gpu, name, longest):
    """What max_seqlen_k says of short requests decides whether a workgroup takes all keys of its rows."""
    case = Paged(**{**SINGLE, **WINDOWS, **TOKENS, **PREFIXES}[name])
    check(_run(gpu, case, max_seqlen_k=longest), case.truth())


@pytest.mark.parametrize("requests", [63, 64, 65, 130])
def test_row_tiles_of_many_requests(gpu, requests):
    """Tiles counted and not, of requests without tokens, with a part of a tile and with several."""
    new = [(0, 3, 17, 64, 65)[(i * 7 + i // 5) % 5] for i in range(requests)]
    case = Paged([n + (i * 13) % 60 for i, n in enumerate(new)], new=new, heads=4, kv_heads=2, head_dim=64, page_size=16)
    check(_run(gpu, case), case.truth())


@pytest.mark.parametrize("dtype", [torch.bfloat16, F16])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2]])
def test_whole_units_of_head_size_64(gpu, new, dtype):
    """Long enough for workgroups of eight waves; 8 and 24 rows."""
    case = Paged([900, 5, 640], new=new, heads=16, kv_heads=2, head_dim=64, page_size=16, dtype=dtype, window=700, n_starting=20)
    check(_run(gpu, case, max_seqlen_q=max(new), max_seqlen_k=900), case.truth())


def test_a_batch_of_thousands(gpu):
    """Requests past the 64 that a wave looks at together, few and none of tokens and keys among them."""
    n = 1500
    case = Paged([(i * 7) % 40 for i in range(n)], new=[i % 3 for i in range(n)], heads=2, kv_heads=1, head_dim=64, page_size=16,
                 prefixes=[i % 50 for i in range(200)], cu_groups=[7 * i + 3 for i in range(201)])
    truth = case.truth()
    for longest_q in (1, 2, 100):
        for longest_k in (48, 5000):
            check(_run(gpu, case, max_seqlen_q=longest_q, max_seqlen_k=longest_k), truth)


@pytest.mark.parametrize("keys", [64, 65])
def test_shares_that_end_with_a_request(gpu, keys):
    """As many requests as workgroups twice over, of the same length: none is cut, or nearly all are."""
    case = Paged([keys] * 1024, heads=2, kv_heads=1, head_dim=64, page_size=16)
    check(_run(gpu, case, max_seqlen_k=5000), case.truth())


def test_more_requests_than_the_kernel_of_few_rows_takes(gpu):
    """Past 65536 requests every one has a row tile of the kernel of rows."""
    n, n_pages = 65600, 4
    k, v = (torch.randn(n_pages, 16, 1, 64, device=gpu).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(n, 1, 64, device=gpu).to(torch.bfloat16)
    table = torch.arange(n, dtype=torch.int32, device=gpu)[:, None] % n_pages
    lens = torch.arange(n, dtype=torch.int32, device=gpu) % 17
    got = paged_cache_attention(q, k, v, table, lens)
    k64, v64 = (x[table[:, 0].long(), :, 0].double() for x in (k, v))
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


@pytest.mark.parametrize("layout", ["apart", "by_head"])
@pytest.mark.parametrize("new", [None, [3, 200]])
def test_layouts_and_strides(gpu, layout, new):
    case = Paged([70, 300], new=new, layout=layout, page_size=32)
    args = case.to(gpu)
    q = torch.empty(len(case.q), case.heads + 4, case.head_dim + 8, dtype=case.dtype, device=gpu)[:, 2:-2, 8:]
    q.copy_(args["q"])
    table = torch.full((2, args["block_table"].shape[1] + 3), -1, dtype=torch.int32, device=gpu)[:, 1:-2]
    table.copy_(args["block_table"])
    store = torch.full((len(case.q), case.heads, 2 * case.head_dim), 7.0, dtype=case.dtype, device=gpu)
    args.update(q=q, block_table=table, out=store[..., : case.head_dim])
    check(paged_cache_attention(**args), case.truth())
    assert (store[..., case.head_dim:] == 7).all()


def test_rows_of_a_table_may_be_one(gpu):
    """Requests that read the same pages, by a table whose rows are one row."""
    case = Paged([200])
    args = case.to(gpu)
    q = torch.randn(3, case.heads, case.head_dim, device=gpu).to(case.dtype)
    args.update(q=q, block_table=args["block_table"].expand(3, -1), seq_lens=args["seq_lens"].expand(3).contiguous())
    got = paged_cache_attention(**args)
    for b in range(3):
        one = paged_cache_attention(**{**args, "q": q[b : b + 1], "block_table": args["block_table"][:1], "seq_lens": args["seq_lens"][:1]})
        assert (got[0][b].float() - one[0][0].float()).abs().max() < 2 * 2.0**-8 * 4 and (got[1][:, b] - one[1][:, 0]).abs().max() < 1e-4


@pytest.mark.parametrize("kind", ["single", "tokens", "window", "prefix"])
def test_entries_that_name_no_page(gpu, kind):
    """Their keys are seen by none, wherever in the row they stand."""
    bad = [(0, 1, lambda n: -1), (1, 0, lambda n: n), (1, 3, lambda n: -(2**31)), (2, 0, lambda n: 2**31 - 1)]
    more = dict(single=dict(), tokens=dict(new=[100, 1, 30]), window=dict(window=70, n_starting=3),
                prefix=dict(prefixes=[200, 90], cu_groups=[0, 1, 3]))[kind]
    if kind == "prefix":
        bad += [(3, 2, lambda n: n + 7), (4, 1, lambda n: -5)]
    case = Paged([300, 333, 30], bad=bad, page_size=32 if kind == "window" else 64, **more)
    check(_run(gpu, case), case.truth())


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("keys", [[100, 9], [9000, 9]])
def test_tokens_of_no_request_are_left(gpu, prefix, keys):
    more = dict(prefixes=[100], cu_groups=[0, 2]) if prefix else {}
    for new in (None, [2, 0]):
        case = Paged(keys, new=new, extra_tokens=5, heads=2, kv_heads=1, **more)
        check(_run(gpu, case, sentinel=3.0), case.truth(), untouched=3.0)


@pytest.mark.parametrize("before", [4, 300])
@pytest.mark.parametrize("new", [[1, 1], [40, 20]])
@pytest.mark.parametrize("prefix", [False, True])
def test_tokens_before_the_first_request_are_left(gpu, before, new, prefix):
    """More of them than a tile of rows holds, too."""
    case = Paged([90, 40], new=new, heads=2, kv_heads=1, **(dict(prefixes=[70], cu_groups=[0, 2]) if prefix else {}))
    args = case.to(gpu)
    q = torch.cat([args["q"].new_zeros(before, 2, 128), args["q"]])
    out, lse = torch.full_like(q, 3.0), torch.full((2, len(q)), 3.0, device=gpu)
    args.update(q=q, cu_seqlens_q=torch.tensor(case.cu + before, dtype=torch.int32, device=gpu), out=out, lse=lse)
    for longest_q in (1, max(new)):
        for longest in (64, 100000):
            (shared_prefix_attention if prefix else paged_cache_attention)(**{**args, "max_seqlen_q": longest_q, "max_seqlen_k": longest})
            assert (out[:before] == 3).all() and (lse[:, :before] == 3).all()
            check((out[before:], lse[:, before:]), case.truth())


def test_no_requests_and_no_pages(gpu):
    case = Paged([10, 20])
    args = case.to(gpu)
    none = {**args, "q": args["q"][:0], "block_table": args["block_table"][:0], "seq_lens": args["seq_lens"][:0]}
    out, lse = paged_cache_attention(**none)
    assert out.shape == (0, 8, 128) and lse.shape == (8, 0)
    empty = {**args, "k_cache": args["k_cache"][:0], "v_cache": args["v_cache"][:0]}
    out, lse = paged_cache_attention(**empty)
    assert (out == 0).all() and (lse == torch.inf).all()


def test_offsets_past_32_bits(gpu):
    """A cache of 10 GB: pages that begin past 2^32 bytes and past 2^31 elements."""
    case = Paged([500, 77], heads=4, kv_heads=2, page_size=64)
    args, n_pages = case.to(gpu), 160_000
    store = torch.empty(n_pages, 64, 2, 2, 128, dtype=case.dtype, device=gpu)
    k, v = store[:, :, 0], store[:, :, 1]
    last = n_pages - case.n_pages
    k[last:], v[last:] = args["k_cache"], args["v_cache"]
    args.update(k_cache=k, v_cache=v, block_table=args["block_table"] + last)
    assert last * k.stride(0) > 2**32
    check(paged_cache_attention(**args), case.truth())


PREFIXES = dict(
    one_group=dict(keys=[1, 2, 33, 64], prefixes=[300], cu_groups=[0, 4]),
    long_prefix=dict(keys=[5, 200, 1, 90], prefixes=[5000], cu_groups=[0, 4], heads=4, kv_heads=1),
    groups=dict(keys=[1 + 7 * i for i in range(11)], prefixes=[64, 700, 17], cu_groups=[0, 2, 9, 11], page_size=32),
    empty_group=dict(keys=[5, 6, 7], prefixes=[64, 100, 17], cu_groups=[0, 2, 2, 3]),
    empty_prefix=dict(keys=[5, 6, 7], prefixes=[0, 100], cu_groups=[0, 2, 3]),
    no_own_keys=dict(keys=[0, 6, 0], prefixes=[80], cu_groups=[0, 3]),
    nothing=dict(keys=[0, 3], prefixes=[0], cu_groups=[0, 2]),
    some_without=dict(keys=[9, 6, 70, 200], prefixes=[90, 30], cu_groups=[1, 2, 3]),
    many=dict(keys=[1 + i % 50 for i in range(150)], prefixes=[500], cu_groups=[0, 150], heads=4, kv_heads=1, head_dim=64),
    many_groups=dict(keys=[1 + i % 9 for i in range(140)], prefixes=[1 + 3 * i for i in range(70)], cu_groups=list(range(0, 141, 2)),
                     heads=2, kv_heads=1, head_dim=64, page_size=16),
    tokens=dict(keys=[9, 40, 200], new=[3, 40, 130], prefixes=[333, 64], cu_groups=[0, 2, 3]),
    no_tokens=dict(keys=[9, 40, 200], new=[3, 0, 130], prefixes=[333, 64], cu_groups=[0, 1, 3], dtype=F16),
    fp16_d64=dict(keys=[9, 40], prefixes=[100], cu_groups=[0, 2], head_dim=64, heads=8, kv_heads=8, dtype=F16),
    group_5=dict(keys=[9, 40, 3], prefixes=[1000], cu_groups=[0, 3], heads=10, kv_heads=2),
)


@pytest.mark.parametrize("name", PREFIXES)
def test_prefixes_against_64_bits(gpu, name):
    case = Paged(**PREFIXES[name])
    check(_run(gpu, case), case.truth())
    check(_run(gpu, case, max_prefix_len=1 << 18, max_seqlen_k=1), case.truth())


def test_a_prefix_gives_what_the_concatenation_gives(gpu):
    """The same keys as a shared prefix and as each request's own first pages."""
    case = Paged([40, 7], prefixes=[128], cu_groups=[0, 2])
    args = case.to(gpu)
    shared = shared_prefix_attention(**args)
    whole = paged_cache_attention(args["q"], args["k_cache"], args["v_cache"],
                                  torch.cat([args["prefix_table"][:, :2].expand(2, -1), args["block_table"]], 1).contiguous(), args["seq_lens"] + 128)
    truth = case.truth()
    check(shared, truth)
    check(whole, truth)


@pytest.mark.parametrize("name", ["long", "mixed", "long_prefix"])
def test_the_same_twice(gpu, name):
    case = Paged(**{**SINGLE, **TOKENS, **PREFIXES}[name])
    first, second = _run(gpu, case), _run(gpu, case)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("prefix", [False, True])
def test_a_callers_workspace_is_enough_and_bounded(gpu, prefix):
    case = Paged([9000, 20], heads=2, kv_heads=1, **(dict(prefixes=[6000], cu_groups=[0, 2]) if prefix else {}))
    args = case.to(gpu)
    n = (shared_prefix_workspace_bytes if prefix else paged_cache_workspace_bytes)(**args)
    call = shared_prefix_attention if prefix else paged_cache_attention
    store = torch.full((n + 4096,), 0xEE, dtype=torch.uint8, device=gpu)
    check(call(**args, workspace=store[:n]), case.truth())
    assert (store[n:] == 0xEE).all()
    with pytest.raises(AssertionError, match="workspace"):
        call(**args, workspace=store[: n - 1])


@pytest.mark.parametrize("prefix", [False, True])
def test_on_another_stream(gpu, prefix):
    case = Paged([900, 20], **(dict(prefixes=[600], cu_groups=[0, 2]) if prefix else {}))
    args, truth = case.to(gpu), case.truth()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = (shared_prefix_attention if prefix else paged_cache_attention)(**args)
    stream.synchronize()
    check(got, truth)


def test_calls_at_the_same_time(gpu):
    """Two streams, and two graphs with a workspace each, replayed side by side."""
    cases = [Paged([3000, 9, 700], heads=4, kv_heads=2), Paged([2500, 30], heads=4, kv_heads=2, prefixes=[3000], cu_groups=[0, 2], seed=1)]
    calls = [(paged_cache_attention, paged_cache_workspace_bytes), (shared_prefix_attention, shared_prefix_workspace_bytes)]
    args, truths, streams = [c.to(gpu) for c in cases], [c.truth() for c in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(calls[i][0](**args[i]))
    torch.cuda.synchronize()
    for results, truth in zip(got, truths):
        for result in results:
            check(result, truth)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for i, graph in enumerate(graphs):
        more = dict(out=torch.empty_like(args[i]["q"]), lse=torch.empty(args[i]["q"].shape[1::-1], device=gpu),
                    workspace=torch.empty(calls[i][1](**args[i]), dtype=torch.uint8, device=gpu))
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=streams[i]):
            calls[i][0](**args[i], **more)
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


@pytest.mark.parametrize("prefix", [False, True])
def test_captured_and_replayed_with_other_lengths(gpu, prefix):
    """One graph for all steps: lengths are read on the device."""
    more = dict(prefixes=[600], cu_groups=[0, 3]) if prefix else {}
    case = Paged([2000, 900, 64], heads=4, kv_heads=2, **more)
    args = case.to(gpu)
    call = shared_prefix_attention if prefix else paged_cache_attention
    call(**args)
    out, lse = torch.empty_like(args["q"]), torch.empty(4, 3, device=gpu)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        call(**args, out=out, lse=lse)
    for lens in ([2000, 900, 64], [1, 0, 64], [1999, 17, 33], [2000, 900, 64]):
        args["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = call(**args)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        torch.cuda.synchronize()


@pytest.mark.parametrize("wrong", ["q_type", "cache_type", "q_axes", "cache_strides", "tables", "lens", "cu", "no_cu", "out", "lse", "dim", "fp32",
                                   "window", "wide_window", "half_a_token", "scale", "page_size", "aligned", "cpu", "heads"])
def test_refusals(gpu, wrong):
    case = Paged([70, 30], head_dim=128)
    args = case.to(gpu)
    q, k, v, table = args["q"], args["k_cache"], args["v_cache"], args["block_table"]
    change = dict(
        q_type=dict(q=q.half()), cache_type=dict(v_cache=v.half()), q_axes=dict(q=q[0]), cache_strides=dict(v_cache=v.contiguous()),
        tables=dict(block_table=table.long()), lens=dict(seq_lens=args["seq_lens"][:1]), cu=dict(cu_seqlens_q=args["seq_lens"]),
        no_cu=dict(q=torch.cat([q, q])), out=dict(out=q[:1].clone()), lse=dict(lse=torch.empty(2, 8, device=gpu)),
        dim=dict(q=q[..., :96].contiguous(), k_cache=k[..., :96], v_cache=v[..., :96]),
        fp32=dict(q=q.float(), k_cache=k.float(), v_cache=v.float()), window=dict(window=0), wide_window=dict(window=1 << 40),
        half_a_token=dict(window=9, n_starting=1.5), scale=dict(softmax_scale=0.0),
        page_size=dict(k_cache=k[:, :40], v_cache=v[:, :40]),
        aligned=dict(q=torch.empty(2 * 8 * 128 + 8, dtype=q.dtype, device=gpu)[4 : 4 + 2 * 8 * 128].view(2, 8, 128)),
        cpu=dict(k_cache=k.cpu(), v_cache=v.cpu()), heads=dict(q=q[:, :5].contiguous()))[wrong]
    with pytest.raises((ValueError, TypeError, AssertionError)):
        paged_cache_attention(**{**args, **change})
