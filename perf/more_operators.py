"""The operators of a paged K/V cache that is held in 4 bits, as they are measured.

Three kinds of case:

* ``write``: a step's keys and values put into the cache through the slot map, and the same rows read back, which is what
  later steps will see of them;
* ``read``: rows of a cache taken out of it again in 16 bits, through a slot map;
* ``attention``: attention over the cache, causal or with a sliding window and first tokens that stay visible.

What the cache holds: every 32 neighbouring elements of a token's key or value share a scale 2^e, and each is one of the 16
numbers +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times that scale.  e is the smallest whole number (of [-127, 127]) for which no element's
size exceeds 7 * 2^e, elements go to the nearest of the numbers that their type can hold, ties to the one of even code.  Bytes of 16
tokens of a head lie together: K's codes token by token, V's in pieces of a sixteenth of a row, those of four tokens side by side,
then the scales' exponents.

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
    case.update(changes)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # One token a request of a mid-sized batch into the cache of an 8B model's layer: latency counts.
        _case("write", "write_decode_64", requests=64, longest=1000, ragged=True),
        # A step's worth of prompts.
        _case("write", "write_prompts_16k", requests=16, longest=1024, new=1024),
        # Ragged prompts in fp16 with small heads and small pages.
        _case("write", "write_ragged_fp16_d64", requests=24, longest=900, new=700, ragged=True, heads=8, kv_heads=8, head_dim=64,
              page_size=16, dtype="fp16"),
        # One conversation's context taken back to 16 bits.
        _case("read", "read_1x1000", longest=1000),
        # Long contexts taken back to 16 bits, to go on with them in a cache of 16 bits.
        _case("read", "read_4x32k", requests=4, longest=32768, page_size=256),
        # One short conversation: latency counts.
        _case("attention", "decode_1x1000", longest=1000),
        # A batch in the middle of its answers: lengths spread over a factor of sixteen.
        _case("attention", "decode_64_ragged_8k", requests=64, longest=8192, ragged=True),
        # A few long contexts: each has to be spread over the whole device.
        _case("attention", "decode_4x128k", requests=4, longest=131072, page_size=256),
        # Sinks and a sliding window over long caches, head size 64, no grouped queries, fp16, small pages.
        _case("attention", "decode_window_fp16_d64", requests=32, longest=16384, ragged=True, heads=8, kv_heads=8, head_dim=64,
              page_size=16, dtype="fp16", window=1000, n_starting=16),
        # Five proposed tokens a request, checked at once: up to 25 rows of a kv head.
        _case("attention", "few_24x5_ragged_4k", requests=24, longest=4000, new=5, ragged=True, heads=40),
        # Prompts in chunks, with the window and the first tokens that lambda_mask_fn has by default.
        _case("attention", "prompt_window_2x2k_of_16k", requests=2, longest=16384, new=2048, window=4096, n_starting=64),
        # Ragged prompts from their start.
        _case("attention", "prompts_ragged_12x1k_fp16", requests=12, longest=1024, new=1024, ragged=True, dtype="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "read", "attention", "attention", "attention"))
    heads, kv_heads = rng.choice(((8, 2), (16, 4), (32, 8), (40, 8), (8, 8)))
    common = dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice((64, 128, 128)), page_size=rng.choice((16, 64, 64, 256)),
                  dtype=rng.choice(("bf16", "bf16", "fp16")), lengths_seed=rng.randrange(1 << 20), ragged=rng.random() < 0.7)
    if kind == "write":
        new = rng.choice((1, _log_uniform(rng, 2, 2048)))
        return _case(kind, requests=_log_uniform(rng, 1, max(1, 16384 // new) if new > 1 else 512), longest=new + _log_uniform(rng, 1, 100),
                     new=new, **common)
    if kind == "read":
        requests = _log_uniform(rng, 1, 64)
        return _case(kind, requests=requests, longest=_log_uniform(rng, 16, 131072 // requests), **common)
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


def _visible(case):
    """``(pairs, keys)``: visible (query, key) pairs, and the keys any query of a request sees."""
    pairs = seen = 0
    for keys, new in zip(*_lengths(case)):
        p = np.arange(keys - new, keys)
        first = np.maximum(0, p - case["window"] + 1) if case["window"] else np.zeros_like(p)
        starting = np.minimum(first, case["n_starting"])
        pairs += int((p + 1 - first + starting).sum())
        seen += int(keys - first[0] + starting[0])
    return pairs, seen


def work(case):
    keys, new = _lengths(case)
    heads, d = case["kv_heads"], case["head_dim"]
    held, wide = heads * d * 17 // 16, heads * d * 4  # bytes of a key and its value: in the cache, in 16 bits
    if case["kind"] == "write":
        return {"bytes": int(new.sum()) * (2 * wide + held + 8), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": int(keys.sum()) * (held + wide + 8), "flops": 0}
    pairs, seen = _visible(case)
    outputs = int(new.sum()) * case["heads"] * (d * 4 + 4)  # q, out and the LSE
    return {"bytes": int(seen * held + outputs), "flops": int(4 * pairs * case["heads"] * d)}


# ---------------------------------------------------------------------------
# the cache's bytes
# ---------------------------------------------------------------------------


def _pieces(cache):
    """Views of a cache ``[pages, heads, blocks, 17 D]``: K's codes ``[.., 16 tokens, D / 2]``, V's ``[.., 4, 16 pieces, 4
    tokens, D / 32]``, K's exponents ``[.., 16 tokens, D / 32]`` and V's ``[.., 4, D / 32, 4 tokens]``."""
    d = cache.shape[3] // 17
    k, v, k_exp, v_exp = cache.split((8 * d, 8 * d, d // 2, d // 2), 3)
    return (k.unflatten(3, (16, d // 2)), v.unflatten(3, (4, 16, 4, d // 32)), k_exp.unflatten(3, (16, d // 32)),
            v_exp.unflatten(3, (4, d // 32, 4)))


def _quantized(x):
    """Codes, two a byte, and exponents' bytes of ``x [..., D]``."""
    largest_e = {torch.bfloat16: 126, torch.float16: 14}[x.dtype]  # of a block with the type's largest number, of which 4 are too many
    x = x.float().unflatten(-1, (-1, 32))
    fraction, exponent = torch.frexp(x.abs().amax(-1))  # fraction in [0.5, 1), of nothing 0
    e = torch.where(fraction == 0, -127, exponent - 3 + (fraction > 0.875)).clamp(min=-127)
    y = x * ((127 - e) << 23).to(torch.int32).view(torch.float32)[..., None]
    size = y.abs()
    size = torch.where((e == largest_e)[..., None], size.clamp(max=3.0), size)
    code = sum((size > a).to(torch.uint8) + (size >= b) for a, b in ((0.25, 0.75), (1.25, 1.75), (2.5, 3.5))) + (size > 5.0)
    code = (code + 8 * (y < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _values(codes, exponents):
    """The numbers in 32 bits that codes ``[..., D / 2]`` and exponents ``[..., D / 32]`` stand for."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    size = code & 7
    level = torch.where(size < 4, 0.5 * size, torch.where(size < 6, size - 2.0, 2.0 * size - 8.0))
    level = torch.where(code > 7, -level, level).unflatten(-1, (-1, 32))
    e = exponents.int()
    scale = torch.where(e == 0, 0x00400000, e << 23).to(torch.int32).view(torch.float32)
    return (level * scale[..., None]).flatten(-2)


def _put(cache, page, offset, k, v):
    """Keys and values ``[n, heads, D]`` into their places."""
    block, j = offset // 16, offset % 16
    k_at, v_at, k_exp, v_exp = _pieces(cache)
    codes, exponents = _quantized(k)
    k_at[page, :, block, j], k_exp[page, :, block, j] = codes, exponents
    codes, exponents = _quantized(v)
    v_at[page, :, block, j // 4, :, j % 4] = codes.unflatten(2, (16, -1))
    v_exp[page, :, block, j // 4, :, j % 4] = exponents


def _taken(cache, page, offset):
    """What ``_put`` has put there, in 32 bits."""
    block, j = offset // 16, offset % 16
    k_at, v_at, k_exp, v_exp = _pieces(cache)
    return (_values(k_at[page, :, block, j], k_exp[page, :, block, j]),
            _values(v_at[page, :, block, j // 4, :, j % 4].flatten(2), v_exp[page, :, block, j // 4, :, j % 4]))


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
    return table


def _filled(n_pages, page_size, heads, d, dtype, generator):
    """A cache of normal keys and values."""
    cache = torch.empty(n_pages, heads, page_size // 16, 17 * d, dtype=torch.uint8, device="cuda")
    k_at, v_at, k_exp, v_exp = _pieces(cache)
    at_once = max(1, (1 << 26) // (page_size * heads * d))
    for begin in range(0, n_pages, at_once):
        some = slice(begin, min(begin + at_once, n_pages))
        shape = (some.stop - begin, heads, page_size // 16, 16, d)
        k_at[some], k_exp[some] = _quantized(_normal(shape, dtype, generator))
        codes, exponents = _quantized(_normal(shape, dtype, generator))
        v_at[some] = codes.view(*shape[:3], 4, 4, 16, d // 32).transpose(4, 5)
        v_exp[some] = exponents.view(*shape[:3], 4, 4, d // 32).transpose(4, 5)
    return cache


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    keys, new = _lengths(case)
    size, dtype, kind = case["page_size"], DTYPES[case["dtype"]], case["kind"]
    tokens, heads, kv_heads, head_dim = int(new.sum()), case["heads"], case["kv_heads"], case["head_dim"]
    n_pages = int((-(-keys // size)).sum()) + 3
    table = _pages_of(keys, size, rng.permutation(n_pages))
    state = dict(case=case, page_size=size, dtype=dtype)
    if kind != "attention":
        # the slots of the requests' new tokens, or of all they have
        count = new if kind == "write" else keys
        ends = np.cumsum(count)
        request = np.repeat(np.arange(len(count)), count)
        position = np.arange(int(ends[-1])) - (ends - count)[request] + (keys - count)[request]
        slots = table[request, position // size] * size + position % size
        state.update(slots=torch.as_tensor(slots, device="cuda"))
    if kind == "write":
        kv = _normal((tokens, 2, kv_heads, head_dim), dtype, generator)  # as a fused projection leaves them
        cache = torch.zeros(n_pages, kv_heads, size // 16, 17 * head_dim, dtype=torch.uint8, device="cuda")
        state.update(k=kv[:, 0], v=kv[:, 1], cache=cache)
        return state
    state.update(cache=_filled(n_pages, size, kv_heads, head_dim, dtype, generator))
    if kind == "attention":
        # scores of standard deviation 2, as trained heads have: neither flat nor a single key
        state.update(q=_normal((tokens, heads, head_dim), dtype, generator, 2.0), table=_i32(table), seq_lens=_i32(keys),
                     cu_q=_i32(np.concatenate([[0], np.cumsum(new)])), longest_q=int(new.max()), longest_k=int(keys.max()),
                     scale=head_dim**-0.5)
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
    from dcp_amd.flash_attn_interface import quantized_cache_attention
    from dcp_amd.ops import quantized_cache_read, quantized_cache_write

    def write(s):
        quantized_cache_write(s["k"], s["v"], s["slots"], s["cache"])
        return quantized_cache_read(s["cache"], s["slots"], s["dtype"])

    def read(s):
        return quantized_cache_read(s["cache"], s["slots"], s["dtype"])

    def attention(s):
        return quantized_cache_attention(s["q"], s["cache"], s["table"], s["seq_lens"], cu_seqlens_q=s["cu_q"],
                                         max_seqlen_q=s["longest_q"], max_seqlen_k=s["longest_k"], window=s["case"]["window"] or None,
                                         n_starting=s["case"]["n_starting"])

    return dict(write=write, read=read, attention=attention)


def _plain_write(s):
    page, offset = s["slots"] // s["page_size"], s["slots"] % s["page_size"]
    _put(s["cache"], page, offset, s["k"], s["v"])
    return tuple(x.to(s["dtype"]) for x in _taken(s["cache"], page, offset))


def _plain_read(s):
    return tuple(x.to(s["dtype"]) for x in _taken(s["cache"], s["slots"] // s["page_size"], s["slots"] % s["page_size"]))


def _rows(q, first, n, longest, kv_heads):
    """Tokens first[b] .. first[b] + n[b] of ``q`` as ``[b, kv head, longest * group, head_dim]`` in 32 bits, zeros behind a
    row's last, and which of them there are."""
    at = torch.arange(longest, device="cuda")
    live = at < n[:, None]
    index = torch.where(live, first[:, None] + at, 0)
    rows = torch.where(live[..., None, None], q.float()[index], 0.0)
    return rows.unflatten(2, (kv_heads, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous(), live


def _gathered(cache, table):
    """The tables' keys and values as ``[b, kv head, key, head_dim]`` in 32 bits."""
    pages = cache[table.long().clamp(min=0)].transpose(1, 2).flatten(2, 3)  # [b, head, block, 17 D]
    k, v, k_exp, v_exp = _pieces(pages)
    v, v_exp = v.transpose(4, 5).flatten(5, 6), v_exp.transpose(4, 5)
    return _values(k, k_exp).flatten(2, 3), _values(v, v_exp).flatten(2, 4)


def _by_token(x, live):
    """``[b, kv head, longest * group, ...]`` back to ``[token, head, ...]``."""
    return x.unflatten(2, (live.shape[1], -1)).transpose(1, 2).flatten(2, 3)[live]


def _plain_attention(s):
    case, first, n = s["case"], s["cu_q"][:-1].long(), s["cu_q"].diff().long()
    q, live = _rows(s["q"], first, n, s["longest_q"], case["kv_heads"])
    k, v = _gathered(s["cache"], s["table"])
    key = torch.arange(k.shape[2], device="cuda")
    at = torch.arange(s["longest_q"], device="cuda").repeat_interleave(case["heads"] // case["kv_heads"])
    p = ((s["seq_lens"].long() - n)[:, None] + at)[:, None, :, None]
    visible = key <= p
    if case["window"]:
        visible &= (key < case["n_starting"]) | (key > p - case["window"])
    scores = torch.where(visible, torch.matmul(q, k.transpose(2, 3)) * s["scale"], -math.inf)
    m = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(m > -math.inf, m, 0.0))
    total = weights.sum(-1, keepdim=True)
    out = torch.where(total > 0, torch.matmul(weights, v) / total, 0.0)
    lse = torch.where(total > 0, m + torch.log(total), math.inf)
    return _by_token(out, live).to(s["q"].dtype), _by_token(lse, live)[..., 0].t().contiguous()


_PLAIN = dict(write=_plain_write, read=_plain_read, attention=_plain_attention)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e, from its bits (a power function may be off by one)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest_held(x):
    """What is held of ``x [..., D]``: the level that is nearest, found by its distance from all."""
    largest = torch.finfo(x.dtype).max
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 2.0**-140) / 7.0))
    e = torch.where(top > 7.0 * _power(e), e + 1, torch.where(top <= 7.0 * _power(e - 1), e - 1, e)).clamp(min=-127)
    scale = _power(e)
    size = x.abs() / scale
    best, off = torch.zeros_like(size), size.clone()
    for code, level in enumerate(_LEVELS[1:], 1):
        d = (size - level).abs()
        closer = ((d < off) | ((d == off) & (code % 2 == 0))) & (level * scale <= largest)
        best, off = torch.where(closer, level, best), torch.where(closer, d, off)
    return (torch.sign(x) * best * scale).flatten(-2)


def _row_held(cache, page, offset):
    """Keys and values of places, ``[n, heads, D]`` each: byte by byte from the layout."""
    d = cache.shape[3] // 17
    element, table = torch.arange(d, device="cuda"), torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), dtype=torch.float64, device="cuda")
    block, j = offset // 16, (offset % 16)[:, None]
    rows = cache[page, :, block]  # [n, heads, 17 D]
    piece = d // 16

    def held(byte, exponent):
        codes = torch.gather(rows, 2, byte[:, None].expand(-1, rows.shape[1], -1)).long()
        codes = (codes >> (4 * (element % 2))) & 15
        e = torch.gather(rows, 2, exponent[:, None].expand(-1, rows.shape[1], -1)).long()
        return table[codes] * _power(e - 127)

    k = held(j * (d // 2) + element // 2, 16 * d + j * (d // 32) + element // 32)
    v = held(8 * d + ((j // 4 * 16 + element // piece) * 4 + j % 4) * (piece // 2) + element % piece // 2,
             16 * d + d // 2 + (j // 4 * (d // 32) + element // 32) * 4 + j % 4)
    return k, v


def exact(case, seed):
    s = prepare(case, seed)
    size = case["page_size"]
    if case["kind"] == "write":
        return _nearest_held(s["k"]), _nearest_held(s["v"])
    if case["kind"] == "read":
        return _row_held(s["cache"], s["slots"] // size, s["slots"] % size)
    keys, new = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[1::-1], dtype=torch.float64, device="cuda")
    begin = 0
    for b in range(len(keys)):
        j = torch.arange(int(keys[b]), device="cuda")
        k, v = _row_held(s["cache"], s["table"][b].long()[j // size], j % size)
        p = torch.arange(int(keys[b] - new[b]), int(keys[b]), device="cuda")[:, None]
        hidden = j > p
        if case["window"]:
            hidden |= (j <= p - case["window"]) & (j >= case["n_starting"])
        for h in range(case["heads"]):
            scores = s["q"][begin : begin + int(new[b]), h].double() @ k[:, h // group].t() * s["scale"]
            scores.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(scores, 1)
            lse[h, begin : begin + int(new[b])] = total
            out[begin : begin + int(new[b]), h] = torch.exp(scores - total[:, None]) @ v[:, h // group]
        begin += int(new[b])
    return out, lse
