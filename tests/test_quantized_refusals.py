"""Arguments that the entry points of a cache in 4 bits refuse before anything is launched, and numbers that they do not hold (CPU: the
addresses are never read)."""

import subprocess
from pathlib import Path

import pytest
import torch

from dcp_amd import _lib
from dcp_amd.flash_attn_interface import _QUANTIZED_ARGS, _quantized_args
from dcp_amd.ops import quantized_cache, quantized_cache_pages, quantized_cache_read, quantized_cache_write

WRITE = dict(k=16, v=16, slots=16, cache=16, n_tokens=3, heads=2, head_dim=64, dtype=0, token=128, head=64, n_pages=4, page_size=16, page=2176,
             cache_head=1088, stream=0)
READ = dict(cache=16, slots=16, **{x: WRITE[x] for x in ("k", "v")}, **{x: WRITE[x] for x in list(WRITE)[4:]})
ATTN = dict(q=16, cache=16, out=16, lse=16, table=16, lens=16, cu=0, q_token=512, q_head=128, out_token=512, out_head=128, page=4352, head=2176, stride=256,
            n_tokens=2, batch=2, heads=4, kv_heads=2, head_dim=128, n_pages=4, page_size=16, width=256, max_q=1, max_k=4096, window=0, n_starting=0,
            dtype=0, scale=1.0)
CALLS = {"dcp_quantized_cache_write": WRITE, "dcp_quantized_cache_read": READ, "attention": ATTN}


def _call(name, **changed):
    workspace, n_bytes = changed.pop("workspace", 16), changed.pop("bytes", 1 << 40)
    values = {**CALLS[name], **changed}.values()
    if name.startswith("dcp"):
        _lib.call(name, *values)
    else:
        _lib.call("dcp_quantized_attn", _QUANTIZED_ARGS.pack(*values), workspace, n_bytes, 0)


@pytest.fixture(scope="module", autouse=True)
def built():
    if not _lib.LIB_PATH.exists():
        from dcp_amd import build

        build.build(verbose=False)


@pytest.mark.parametrize("name,wrong,message", [
    *[(name, wrong, message) for name in ("dcp_quantized_cache_write", "dcp_quantized_cache_read") for wrong, message in (
        (dict(dtype=2), "bf16 and fp16"), (dict(dtype=-1), "bf16 and fp16"), (dict(head_dim=96), "head_dim"), (dict(head_dim=32), "head_dim"),
        (dict(n_tokens=-1), "sizes"), (dict(heads=0), "sizes"), (dict(n_pages=-1), "sizes"), (dict(page_size=0), "multiple of 16"),
        (dict(page_size=24), "multiple of 16"), (dict(token=-128), "multiples of 8"), (dict(head=4), "multiples of 8"), (dict(page=-2176), "multiples of 16"),
        (dict(page=2168), "multiples of 16"), (dict(cache_head=8), "multiples of 16"), (dict(heads=1 << 21), "too many heads"),
        (dict(n_pages=1 << 60), "too many pages"), (dict(n_tokens=2**31 - 1, heads=1 << 12), "too many rows"), (dict(k=0), "null"), (dict(v=0), "null"),
        (dict(slots=0), "null"), (dict(cache=0), "null"), (dict(k=24), "aligned"), (dict(v=18), "aligned"), (dict(cache=8), "aligned"))],
    *[("attention", wrong, message) for wrong, message in (
        (dict(dtype=2), "bf16 and fp16"), (dict(dtype=9), "bf16 and fp16"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
        (dict(heads=5), "multiple of n_heads_kv"), (dict(kv_heads=0), "multiple of n_heads_kv"), (dict(n_tokens=-1), "negative size"),
        (dict(batch=-1), "negative size"), (dict(n_pages=-1), "negative size"), (dict(scale=0.0), "softmax_scale"),
        (dict(scale=float("nan")), "softmax_scale"), (dict(page_size=24), "multiple of 16"), (dict(page_size=0), "multiple of 16"),
        (dict(width=0), "empty block table"), (dict(stride=-4), "empty block table"), (dict(width=1 << 27), "too many keys"),
        (dict(head=2184), "multiples of 8"), (dict(q_head=4), "multiples of 8"), (dict(out_head=2), "multiples of 8"), (dict(page=-4352), "negative stride"),
        (dict(out_token=0), "negative stride"), (dict(q=24), "aligned"), (dict(out=8), "aligned"), (dict(cache=8), "aligned"),
        (dict(n_tokens=1 << 30, cu=16), "too many queries"), (dict(n_tokens=3), "one token"), (dict(lse=0), "null"), (dict(table=0), "null"),
        (dict(lens=0), "null"), (dict(cache=0), "null"), (dict(max_q=0), "longest"), (dict(max_k=-1), "longest"), (dict(window=-1), "window"),
        (dict(n_starting=-1), "window"), (dict(bytes=64), "workspace"), (dict(workspace=8), "workspace"), (dict(workspace=0), "workspace"))],
])
def test_refused(name, wrong, message):
    error = ValueError if message in ("bf16 and fp16", "head_dim") else AssertionError
    with pytest.raises(error, match=message):
        _call(name, **wrong)


@pytest.mark.parametrize("name,empty", [
    ("dcp_quantized_cache_write", dict(n_tokens=0, k=0, v=0, slots=0)), ("dcp_quantized_cache_write", dict(n_pages=0, cache=0)),
    ("dcp_quantized_cache_read", dict(n_tokens=0, k=0, v=0, slots=0, cache=0)),
    ("attention", dict(n_tokens=0, batch=0, q=0, out=0, lse=0)), ("attention", dict(n_tokens=0, cu=16)),
])
def test_nothing_to_do(name, empty):
    _call(name, **empty)


def test_workspaces_are_none_for_nothing_and_more_for_more():
    lib = _lib.load()
    size = lambda **changed: lib.dcp_quantized_attn_workspace_bytes(_QUANTIZED_ARGS.pack(*{**ATTN, **changed}.values()))
    assert lib.dcp_quantized_attn_workspace_bytes(None) == 0 and size(n_tokens=0, batch=0) == 0 and size(head_dim=96) == 0
    assert 0 < size() < size(max_q=16)
    with pytest.raises(AssertionError, match="null"):
        _lib.call("dcp_quantized_attn", None, 0, 0, 0)


def test_the_arguments_have_the_size_the_library_takes(tmp_path):
    (tmp_path / "size.cpp").write_text('#include <stddef.h>\n#include "dcp_hip.h"\nstatic_assert(sizeof(dcp_quantized_attn_args) == %d, "");\n'
                                       'static_assert(offsetof(dcp_quantized_attn_args, softmax_scale) == %d, "");\n'
                                       % (_QUANTIZED_ARGS.size, _QUANTIZED_ARGS.size - 4))
    subprocess.run(["g++", "-fsyntax-only", f"-I{Path(__file__).resolve().parents[1] / 'include'}", str(tmp_path / "size.cpp")], check=True)


@pytest.fixture
def here(monkeypatch):
    """Tensors without memory on "the current device", and the calls that would have been made."""
    calls = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: torch.empty(0, device="meta").get_device())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0)
    monkeypatch.setattr(quantized_cache._lib, "call", lambda *args: calls.append(args))
    return calls


def _empty(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("sizes", [dict(n_tokens=2**32 + 3), dict(heads=2**32 + 2), dict(tiles=2**28 + 1)])
def test_sizes_that_32_bits_do_not_hold(here, sizes):
    n, heads, tiles = (sizes.get(name, 2) for name in ("n_tokens", "heads", "tiles"))
    x, slots, cache = _empty(n, heads, 64), _empty(n, dtype=torch.int64), _empty(3, heads, tiles, 17 * 64, dtype=torch.uint8)
    for call in (lambda: quantized_cache_write(x, x, slots, cache), lambda: quantized_cache_read(cache, slots, out=(x, x))):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    q, table = _empty(2, 4 * heads, 64), _empty(2, 3, dtype=torch.int32)
    if n == 2:
        with pytest.raises(ValueError, match="32 bits"):
            _quantized_args(q, cache, table, _empty(2, dtype=torch.int32), None, None, None, None, None, 0, q, _empty(4 * heads, 2, dtype=torch.float32))
    assert not here


def test_sizes_that_fit(here):
    x, cache = _empty(2, 2, 64), _empty(2**33, 2, 2, 17 * 64, dtype=torch.uint8)  # (pages are counted in 64 bits)
    quantized_cache_write(x, x, _empty(2, dtype=torch.int64), cache)
    quantized_cache_read(cache, _empty(2, dtype=torch.int64), out=(x, x))
    assert [call[0] for call in here] == ["dcp_quantized_cache_write", "dcp_quantized_cache_read"] and here[0][11] == here[1][11] == 2**33


@pytest.mark.parametrize("scale", [1e39, -1e39, "half"])
def test_a_scale_that_32_bits_do_not_hold(here, scale):
    q, cache, i32 = _empty(2, 4, 64), _empty(3, 2, 1, 17 * 64, dtype=torch.uint8), torch.int32
    with pytest.raises(ValueError, match="softmax_scale"):
        _quantized_args(q, cache, _empty(2, 3, dtype=i32), _empty(2, dtype=i32), None, None, None, scale, None, 0, None, None)


@pytest.mark.parametrize("wrong", [(4, 24, 2, 64), (4, 0, 2, 64), (4, -16, 2, 64), (4, 16, 2, 96), (4, 16, 2, 256)])
def test_pages_of_other_shapes(wrong):
    with pytest.raises(ValueError):
        quantized_cache_pages(*wrong, device="cpu")
    assert quantized_cache_pages(4, 48, 2, 64, device="cpu").shape == (4, 2, 3, 17 * 64)
