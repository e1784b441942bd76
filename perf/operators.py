"""The operators that answer over a paged cache, as they are measured.

Four kinds of case, each a call of one public entry point:

* ``tables``: the block tables and the slot map of one step, from the requests' lengths;
* ``write``: the step's keys and values put into the cache through the slot map;
* ``attention``: attention over the cache, causal or with a sliding window and first tokens that stay visible;
* ``prefix``: attention of a batch whose requests share long prefixes.

``own`` says which form ``run`` takes: the plain one of elementary torch operations, or the framework's entry points.
A case holds numbers and names only; lengths follow from its ``lengths_seed``.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(kind, name=None, **changes):
    case = dict(kind=kind, requests=1, longest=1024, ragged=False, new=1, heads=32, kv_heads=8, head_dim=128, page_size=64,
                dtype="bf16", lengths_seed=0)
    if kind == "attention":
        case.update(window=0, n_starting=0)  # window 0: all keys up to the query's own
    if kind == "prefix":
        case.update(prefix=8192, groups=1)
    case.update(changes)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # A decoding step of a mid-sized batch: one token a request; a launch and little else.
        _case("tables", "tables_decode_64", requests=64, longest=8192, ragged=True),
        # Prompts admitted together, up to 1024 tokens each: the slot map is most of it.
        _case("tables", "tables_prompts_256", requests=256, longest=1024, ragged=True, new=1024),
        # One token a request into the cache of an 8B model's layer.
        _case("write", "write_decode_64", requests=64, longest=1000, ragged=True),
        # A step's worth of prompts.
        _case("write", "write_prompts_16k", requests=16, longest=1024, new=1024),
        # One short conversation: latency counts.
        _case("attention", "decode_1x1000", longest=1000),
        # A batch in the middle of its answers: lengths spread over a factor of sixteen.
        _case("attention", "decode_64_ragged_8k", requests=64, longest=8192, ragged=True),
        # A few long contexts: each has to be spread over the whole device.
        _case("attention", "decode_4x128k", requests=4, longest=131072, page_size=256),
        # Sinks and a sliding window over long caches, head size 64, no grouped queries, fp16, small pages.
        _case("attention", "decode_window_fp16_d64", requests=32, longest=16384, ragged=True, heads=8, kv_heads=8, head_dim=64,
              page_size=16, dtype="fp16", window=1000, n_starting=16),
        # Prompts in chunks, with the window and the first tokens that lambda_mask_fn has by default.
        _case("attention", "prompt_window_2x2k_of_16k", requests=2, longest=16384, new=2048, window=4096, n_starting=64),
        # A handful of answers to one question.
        _case("prefix", "prefix_4_of_2k", requests=4, longest=50, ragged=True, prefix=2000),
        # Many samples of one long context.
        _case("prefix", "prefix_64_of_32k", requests=64, longest=1024, ragged=True, prefix=32768),
        # Several shared contexts in one batch, eight q heads of which four share a kv head.
        _case("prefix", "prefix_4_groups_96_of_8k", requests=96, longest=500, ragged=True, prefix=8192, groups=4, heads=8,
              kv_heads=2),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("tables", "write", "attention", "attention", "attention", "prefix", "prefix"))
    heads, kv_heads = rng.choice(((8, 2), (16, 4), (32, 8), (40, 8), (8, 8)))
    common = dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice((64, 128, 128)), page_size=rng.choice((16, 64, 64, 256)),
                  dtype=rng.choice(("bf16", "bf16", "fp16")), lengths_seed=rng.randrange(1 << 20), ragged=rng.random() < 0.7)
    if kind == "tables":
        new = rng.choice((1, 1, _log_uniform(rng, 2, 1024)))
        longest = new + _log_uniform(rng, 1, 16384)
        return _case(kind, requests=_log_uniform(rng, 1, 256 if new > 1 else 4096), longest=longest, new=new, **common)
    if kind == "write":
        new = rng.choice((1, _log_uniform(rng, 2, 2048)))
        return _case(kind, requests=_log_uniform(rng, 1, max(1, 16384 // new) if new > 1 else 512), longest=new + _log_uniform(rng, 1, 100),
                     new=new, **common)
    if kind == "prefix":
        requests = _log_uniform(rng, 1, 96)
        return _case(kind, requests=requests, longest=_log_uniform(rng, 1, 1024), prefix=_log_uniform(rng, 256, 32768 if requests <= 64 else 16384),
                     groups=rng.choice((1, 1, min(requests, 3))), **common)
    requests = _log_uniform(rng, 1, 128)
    longest = _log_uniform(rng, 16, min(131072, 500_000 // requests))
    window = rng.choice((0, 0, _log_uniform(rng, 16, 4096)))
    case = _case(kind, requests=requests, longest=longest, window=window, n_starting=rng.choice((0, 1, 4, 64)) if window else 0, **common)
    if rng.random() < 0.3:  # a few tokens each, or prompts
        most = max(1, min(longest, 2048, 12_000_000 // (requests * longest)))
        case.update(new=rng.choice((min(most, 4), _log_uniform(rng, 1, most))))
    return case


# ---------------------------------------------------------------------------
# what a case's numbers stand for
# ---------------------------------------------------------------------------


def _lengths(case):
    """``(keys, new)`` of every request, the new tokens' keys among them: ``longest`` and ``new`` for all, or spread
    evenly over the logarithm from a sixteenth up, the first request having the most."""
    n, rng = case["requests"], np.random.default_rng(case["lengths_seed"])

    def spread(most):
        low = max(1, most // 16)
        lengths = np.exp(rng.uniform(math.log(low), math.log(most + 1), n)).astype(np.int64).clip(low, most)
        lengths[0] = most
        return lengths

    if not case["ragged"]:
        return np.full(n, case["longest"]), np.full(n, case["new"])
    keys, new = spread(case["longest"]), spread(case["new"])
    return np.maximum(keys, new), new


def _groups(case):
    """Where each group's requests begin, and the last one's end: unequal groups."""
    n, g = case["requests"], case.get("groups", 1)
    return np.array([i * n // g if i % 2 == 0 or g == 1 else (2 * i + 1) * n // (2 * g) for i in range(g)] + [n])


def _prefix_lengths(case):
    """The first prefix in full, each later one an eighth shorter than the one before."""
    return np.array([max(1, int(case["prefix"] * (7 / 8) ** i)) for i in range(case["groups"])])


def _visible(case):
    """``(pairs, keys)``: visible (query, key) pairs of the requests' own keys, and the keys any query of a request sees."""
    pairs = seen = 0
    for keys, new in zip(*_lengths(case)):
        p = np.arange(keys - new, keys)
        first = np.maximum(0, p - case["window"] + 1) if case.get("window") else np.zeros_like(p)
        starting = np.minimum(first, case.get("n_starting", 0))
        pairs += int((p + 1 - first + starting).sum())
        seen += int(keys - first[0] + starting[0])
    return pairs, seen


def work(case):
    keys, new = _lengths(case)
    tokens, size = int(new.sum()), case["kv_heads"] * case["head_dim"] * 4  # bytes of a key and its value
    pages = -(-keys // case["page_size"]) - -(-(keys - new) // case["page_size"])
    if case["kind"] == "tables":
        return {"bytes": int(len(keys) * 16 + tokens * 12 + pages.sum() * 8), "flops": 0}
    if case["kind"] == "write":
        return {"bytes": tokens * (2 * size + 8), "flops": 0}
    pairs, seen = _visible(case)
    if case["kind"] == "prefix":
        ends, prefix = _groups(case), _prefix_lengths(case)
        group_tokens = [new[a:b].sum() for a, b in zip(ends, ends[1:])]
        pairs += int(np.dot(group_tokens, prefix))
        seen += int(prefix[[n > 0 for n in group_tokens]].sum())
    outputs = tokens * case["heads"] * (case["head_dim"] * 4 + 4)  # q, out and the LSE
    return {"bytes": int(seen * size + outputs), "flops": int(4 * pairs * case["heads"] * case["head_dim"])}


# ---------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------


def _normal(shape, dtype, generator, scale=1.0):
    return torch.randn(shape, device="cuda", dtype=torch.float32, generator=generator).mul_(scale).to(dtype)


def _i32(values):
    return torch.as_tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _pages_of(lengths, page_size, pages):
    """A table of one row per length whose pages are the next of ``pages``; -1 behind a row's last."""
    counts = -(-np.asarray(lengths) // page_size)
    table = np.full((len(counts), max(1, int(counts.max()))), -1)
    table[np.arange(table.shape[1])[None] < counts[:, None]] = pages[: counts.sum()]
    return table, pages[counts.sum():]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    keys, new = _lengths(case)
    size, dtype = case["page_size"], DTYPES[case["dtype"]]
    tokens, heads, kv_heads, head_dim = int(new.sum()), case["heads"], case["kv_heads"], case["head_dim"]
    state = dict(case=case, tokens=tokens, page_size=size)
    own_pages = int((-(-keys // size)).sum())
    if case["kind"] == "tables":
        # the pages of what is cached are anywhere in the cache, the free ones as they were given back
        pages = rng.permutation(own_pages + 100)
        table, rest = _pages_of(keys - new, size, pages)
        wide = np.full((len(keys), -(-case["longest"] // size)), -1)
        wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
        state.update(cached=_i32(keys - new), new=_i32(new), table=_i32(wide), free=_i32(rest))
        return state
    prefix = _prefix_lengths(case) if case["kind"] == "prefix" else np.array([], dtype=np.int64)
    n_pages = own_pages + int((-(-prefix // size)).sum()) + 3
    pages = rng.permutation(n_pages)
    table, pages = _pages_of(keys, size, pages)
    cache = _normal((n_pages, size, 2, kv_heads, head_dim), dtype, generator)
    cu = np.concatenate([[0], np.cumsum(new)])
    state.update(kv=cache, k_cache=cache[:, :, 0], v_cache=cache[:, :, 1])
    if case["kind"] == "write":
        request = np.repeat(np.arange(len(new)), new)
        position = np.arange(tokens) - cu[request] + (keys - new)[request]
        slots = table[request, position // size] * size + position % size
        kv = _normal((tokens, 2, kv_heads, head_dim), dtype, generator)  # as a fused projection leaves them
        state.update(k=kv[:, 0], v=kv[:, 1], slots=torch.as_tensor(slots, device="cuda"))
        return state
    # scores of standard deviation 2, as trained heads have: neither flat nor a single key
    state.update(q=_normal((tokens, heads, head_dim), dtype, generator, 2.0), table=_i32(table), seq_lens=_i32(keys),
                 cu_q=_i32(cu), longest_q=int(new.max()), longest_k=int(keys.max()), scale=head_dim**-0.5)
    if case["kind"] == "prefix":
        ends = _groups(case)
        state.update(prefix_table=_i32(_pages_of(prefix, size, pages)[0]), prefix_lens=_i32(prefix), cu_groups=_i32(ends),
                     longest_prefix=int(prefix.max()), longest_group=int(max(cu[b] - cu[a] for a, b in zip(ends, ends[1:]))))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    if own:
        return _own_forms()[state["case"]["kind"]](state)
    return _PLAIN[state["case"]["kind"]](state)


@functools.cache
def _own_forms():
    from dcp_amd.flash_attn_interface import paged_cache_attention, shared_prefix_attention
    from dcp_amd.ops import paged_cache_tables, paged_cache_write

    def tables(s):
        made = paged_cache_tables(s["cached"], s["new"], s["table"], s["free"], s["page_size"], s["tokens"])
        return [made.slot_mapping, made.positions, made.cu_seqlens, made.seq_lens, made.pages_taken, s["table"]]

    def write(s):
        paged_cache_write(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
        return s["kv"]

    def attention(s):
        return paged_cache_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], cu_seqlens_q=s["cu_q"],
                                     max_seqlen_q=s["longest_q"], max_seqlen_k=s["longest_k"], window=s["case"]["window"] or None,
                                     n_starting=s["case"]["n_starting"])

    def prefix(s):
        return shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], s["prefix_lens"], s["cu_groups"],
                                       s["table"], s["seq_lens"], cu_seqlens_q=s["cu_q"], max_seqlen_q=s["longest_q"],
                                       max_seqlen_k=s["longest_k"], max_prefix_len=s["longest_prefix"])

    return dict(tables=tables, write=write, attention=attention, prefix=prefix)


def _plain_tables(s):
    size, table, free = s["page_size"], s["table"], s["free"]
    cached, new = s["cached"].long(), s["new"].long()
    column = torch.arange(table.shape[1], device="cuda")
    have, want = (cached + size - 1) // size, (cached + new + size - 1) // size
    taken = torch.cumsum(want - have, 0)
    fresh = (column >= have[:, None]) & (column < want[:, None])
    index = (taken - want)[:, None] + column  # of the free list
    pages = torch.where(index < free.numel(), free[index.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, pages, table))
    ends = torch.cumsum(new, 0)
    cu = torch.cat([ends.new_zeros(1), ends]).int()
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(ends, token, right=True)
    position = cached[request] + token - (ends - new)[request]
    page = table[request, position // size].long()
    slots = torch.where(page >= 0, page * size + position % size, -1)
    return [slots, position.int(), cu, (cached + new).int(), taken[-1:].int(), table]


def _plain_write(s):
    page, offset = s["slots"] // s["page_size"], s["slots"] % s["page_size"]
    s["k_cache"][page, offset] = s["k"]
    s["v_cache"][page, offset] = s["v"]
    return s["kv"]


def _rows(q, first, n, longest, kv_heads):
    """Tokens first[b] .. first[b] + n[b] of ``q`` as ``[b, kv head, longest * group, head_dim]`` in 32 bits, zeros behind a
    row's last, and where they came from."""
    at = torch.arange(longest, device="cuda")
    live = at < n[:, None]
    index = torch.where(live, first[:, None] + at, 0)
    rows = torch.where(live[..., None, None], q.float()[index], 0.0)
    rows = rows.unflatten(2, (kv_heads, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return rows.contiguous(), live, index


def _gathered(cache, table):
    """The tables' keys or values as ``[b, kv head, key, head_dim]`` in 32 bits."""
    pages = cache[table.long().clamp(min=0)].flatten(1, 2)
    return pages.transpose(1, 2).float().contiguous()


def _by_token(x, live, heads):
    """``[b, kv head, longest * group, ...]`` back to ``[token, head, ...]``."""
    x = x.unflatten(2, (live.shape[1], -1)).transpose(1, 2).flatten(2, 3)
    return x[live]


def _softmax_parts(q, k, v, visible, scale):
    """Row maxima, sums and products of one set of keys; a row that sees none has a sum of zero."""
    s = torch.where(visible, torch.matmul(q, k.transpose(2, 3)) * scale, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _own_keys(s, q, n, longest, case):
    """What the requests' own keys add."""
    k = _gathered(s["k_cache"], s["table"])
    v = _gathered(s["v_cache"], s["table"])
    key = torch.arange(k.shape[2], device="cuda")
    at = torch.arange(longest, device="cuda").repeat_interleave(case["heads"] // case["kv_heads"])
    p = (s["seq_lens"].long() - n)[:, None] + at
    p = p[:, None, :, None]
    visible = key <= p
    if case.get("window"):
        visible &= (key < case["n_starting"]) | (key > p - case["window"])
    return _softmax_parts(q, k, v, visible, s["scale"])


def _plain_attention(s):
    case, first, n = s["case"], s["cu_q"][:-1].long(), s["cu_q"].diff().long()
    q, live, _ = _rows(s["q"], first, n, s["longest_q"], case["kv_heads"])
    m, l, o = _own_keys(s, q, n, s["longest_q"], case)
    out = _by_token(torch.where(l > 0, o / l, 0.0), live, case["heads"]).to(s["q"].dtype)
    lse = _by_token(torch.where(l > 0, m + torch.log(l), math.inf), live, case["heads"])
    return out, lse[..., 0].t().contiguous()


def _plain_prefix(s):
    case, first, n = s["case"], s["cu_q"][:-1].long(), s["cu_q"].diff().long()
    q, live, _ = _rows(s["q"], first, n, s["longest_q"], case["kv_heads"])
    parts = [[_by_token(x, live, case["heads"]) for x in _own_keys(s, q, n, s["longest_q"], case)]]
    ends = s["cu_q"].long()[s["cu_groups"].long()]
    q, live, _ = _rows(s["q"], ends[:-1], ends.diff(), s["longest_group"], case["kv_heads"])
    k, v = _gathered(s["k_cache"], s["prefix_table"]), _gathered(s["v_cache"], s["prefix_table"])
    visible = (torch.arange(k.shape[2], device="cuda") < s["prefix_lens"][:, None])[:, None, None, :]
    parts.append([_by_token(x, live, case["heads"]) for x in _softmax_parts(q, k, v, visible, s["scale"])])
    (m0, l0, o0), (m1, l1, o1) = parts
    m = torch.maximum(m0, m1)
    w0, w1 = torch.exp(m0 - m), torch.exp(m1 - m)
    l = w0 * l0 + w1 * l1
    out = ((w0 * o0 + w1 * o1) / l).to(s["q"].dtype)
    return out, (m + torch.log(l))[..., 0].t().contiguous()


_PLAIN = dict(tables=_plain_tables, write=_plain_write, attention=_plain_attention, prefix=_plain_prefix)


# ---------------------------------------------------------------------------
# the definition in 64 bits, one request after the other
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    size, group = case["page_size"], case["heads"] // case["kv_heads"]
    if case["kind"] == "write":
        flat = s["kv"].flatten(0, 1).double()
        for t, slot in enumerate(s["slots"].tolist()):
            flat[slot, 0], flat[slot, 1] = s["k"][t].double(), s["v"][t].double()
        return flat.view_as(s["kv"])
    keys, new = _lengths(case)
    ends = _groups(case) if case["kind"] == "prefix" else None
    prefix = _prefix_lengths(case) if case["kind"] == "prefix" else None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[1::-1], dtype=torch.float64, device="cuda")

    def rows_of(table, length):
        position = torch.arange(length, device="cuda")
        page = table.long()[position // size]
        return s["kv"][page, position % size].double()  # [key, 2, kv head, head_dim]

    begin, held, held_group = 0, None, None
    for b in range(len(keys)):
        kv, before = rows_of(s["table"][b], int(keys[b])), 0
        if prefix is not None:
            g = int(np.searchsorted(ends, b, side="right")) - 1
            if held_group != g:
                held, held_group = rows_of(s["prefix_table"][g], int(prefix[g])), g
            kv, before = torch.cat([held, kv]), int(prefix[g])
        j = torch.arange(kv.shape[0], device="cuda")
        p = before + torch.arange(int(keys[b] - new[b]), int(keys[b]), device="cuda")[:, None]
        hidden = j > p
        if case.get("window"):
            hidden |= (j <= p - case["window"]) & (j >= case["n_starting"])
        for h in range(case["heads"]):
            scores = s["q"][begin : begin + int(new[b]), h].double() @ kv[:, 0, h // group].t() * s["scale"]
            scores.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(scores, 1)
            lse[h, begin : begin + int(new[b])] = total
            out[begin : begin + int(new[b]), h] = torch.exp(scores - total[:, None]) @ kv[:, 1, h // group]
        begin += int(new[b])
    return out, lse
