"""Arguments that the entry points of the paged cache refuse before anything is launched (CPU: the addresses are never read)."""

import subprocess
from pathlib import Path

import pytest

from dcp_amd import _lib
from dcp_amd.flash_attn_interface import _PAGED_ARGS

TABLES = dict(cached=16, new=16, table=256, stride=4, free=32, slots=512, positions=512, cu=512, lens=512, taken=512, batch=2, width=4, n_free=3,
              page_size=16, n_tokens=5, stream=0)
WRITE = dict(k=16, v=16, slots=16, k_cache=16, v_cache=16, n_tokens=3, heads=2, head_dim=64, elem=2, token=128, head=64, n_pages=4,
             page_size=16, page=2048, cache_token=128, cache_head=64, stream=0)
ATTN = dict(q=16, k=16, v=16, out=16, lse=16, table=16, lens=16, cu=0, prefix_table=0, prefix_lens=0, groups=0, q_token=512, q_head=128, out_token=512,
            out_head=128, page=4096, token=256, head=128, stride=256, prefix_stride=0, n_tokens=2, batch=2, heads=4, kv_heads=2, head_dim=128, n_pages=4,
            page_size=16, width=256, prefix_width=0, n_prefixes=0, max_q=1, max_k=4096, max_prefix=0, window=0, n_starting=0, dtype=0, scale=1.0)
PREFIX = dict(ATTN, prefix_table=16, prefix_lens=16, groups=16, prefix_stride=4, prefix_width=4, n_prefixes=1, max_prefix=64)
CALLS = {"dcp_paged_cache_tables": TABLES, "dcp_paged_cache_write": WRITE, "attention": ATTN, "prefix": PREFIX}


def _call(name, **changed):
    workspace, n_bytes = changed.pop("workspace", 16), changed.pop("bytes", 1 << 40)
    values = {**CALLS[name], **changed}.values()
    if name.startswith("dcp"):
        _lib.call(name, *values)
    else:
        _lib.call("dcp_paged_attn", _PAGED_ARGS.pack(*values), workspace, n_bytes, 0)


@pytest.fixture(scope="module", autouse=True)
def built():
    if not _lib.LIB_PATH.exists():
        from dcp_amd import build

        build.build(verbose=False)


@pytest.mark.parametrize("name,wrong,message", [
    ("dcp_paged_cache_tables", dict(batch=-1), "negative size"),
    ("dcp_paged_cache_tables", dict(n_tokens=-1), "negative size"),
    ("dcp_paged_cache_tables", dict(n_free=-2), "negative size"),
    ("dcp_paged_cache_tables", dict(page_size=0), "page_size"),
    ("dcp_paged_cache_tables", dict(width=0), "do not make a table"),
    ("dcp_paged_cache_tables", dict(stride=3), "do not make a table"),
    *[("dcp_paged_cache_tables", {x: 0}, "null") for x in ("cached", "new", "table", "free", "slots", "positions", "cu", "lens", "taken")],
    *[("dcp_paged_cache_tables", {a: 4096, b: 4100}, "also written") for a in ("cached", "new", "free") for b in ("lens", "cu", "slots", "positions", "table")],
    ("dcp_paged_cache_tables", dict(free=4096, taken=4104), "also written"),
    ("dcp_paged_cache_write", dict(elem=8), "element size"),
    ("dcp_paged_cache_write", dict(n_tokens=-1), "sizes"),
    ("dcp_paged_cache_write", dict(heads=0), "sizes"),
    ("dcp_paged_cache_write", dict(page_size=0), "sizes"),
    ("dcp_paged_cache_write", dict(n_pages=-1), "sizes"),
    ("dcp_paged_cache_write", dict(cache_token=-8), "negative stride"),
    *[("dcp_paged_cache_write", {x: 0}, "null") for x in ("k", "v", "slots", "k_cache", "v_cache")],
    *[(name, wrong, message) for name in ("attention", "prefix") for wrong, message in (
        (dict(dtype=2), "bf16 and fp16"), (dict(dtype=9), "bf16 and fp16"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
        (dict(heads=5), "multiple of n_heads_kv"), (dict(kv_heads=0), "multiple of n_heads_kv"), (dict(n_tokens=-1), "negative size"),
        (dict(batch=-1), "negative size"), (dict(n_pages=-1), "negative size"), (dict(scale=0.0), "softmax_scale"),
        (dict(scale=float("nan")), "softmax_scale"), (dict(page_size=24), "multiple of 16"), (dict(page_size=0), "multiple of 16"),
        (dict(width=0), "empty block tables"), (dict(stride=-4), "empty block tables"), (dict(width=1 << 27), "too many keys"),
        (dict(token=257), "multiples of 8"), (dict(out_head=2), "multiples of 8"), (dict(page=-4096), "negative stride"),
        (dict(out_token=0), "negative stride"), (dict(q=24), "aligned"), (dict(out=8), "aligned"), (dict(k=18), "aligned"),
        (dict(n_tokens=1 << 30, cu=16), "too many queries"), (dict(n_tokens=3), "one token"), (dict(lse=0), "null"), (dict(table=0), "null"),
        (dict(lens=0), "null"), (dict(v=0), "null"), (dict(max_q=0), "longest"), (dict(max_k=-1), "longest"))],
    ("attention", dict(window=-1), "window"),
    ("attention", dict(n_starting=-1), "window"),
    ("attention", dict(bytes=64), "workspace"),
    ("attention", dict(workspace=8), "workspace"),
    ("prefix", dict(n_prefixes=-1), "negative size"),
    ("prefix", dict(window=9), "no window"),
    ("prefix", dict(prefix_width=0), "empty block tables"),
    ("prefix", dict(prefix_table=0), "null"),
    ("prefix", dict(prefix_lens=0), "null"),
    ("prefix", dict(groups=0), "null"),
    ("prefix", dict(max_prefix=0), "longest"),
    ("prefix", dict(bytes=64), "workspace"),
    ("prefix", dict(workspace=0), "workspace"),
])
def test_refused(name, wrong, message):
    error = ValueError if message in ("bf16 and fp16", "head_dim") else AssertionError
    with pytest.raises(error, match=message):
        _call(name, **wrong)


@pytest.mark.parametrize("name,empty", [
    ("dcp_paged_cache_write", dict(n_tokens=0, k=0, v=0, slots=0)), ("dcp_paged_cache_write", dict(n_pages=0, k_cache=0, v_cache=0)),
    ("attention", dict(n_tokens=0, batch=0, q=0, out=0, lse=0)), ("attention", dict(n_tokens=0, cu=16)),
    ("prefix", dict(n_tokens=0, batch=0, n_prefixes=0)),
])
def test_nothing_to_do(name, empty):
    _call(name, **empty)


def test_workspaces_are_none_for_nothing_and_more_for_more():
    lib = _lib.load()
    size = lambda name, **changed: lib.dcp_paged_attn_workspace_bytes(_PAGED_ARGS.pack(*{**CALLS[name], **changed}.values()))
    assert lib.dcp_paged_attn_workspace_bytes(None) == 0 and size("attention", n_tokens=0, batch=0) == 0 and size("attention", head_dim=96) == 0
    assert 0 < size("attention") < size("attention", max_q=16) and size("attention") < size("prefix") < size("prefix", max_k=1 << 20, width=1 << 16)
    # prompts of many rows need none: no share of the keys to join
    assert size("attention", n_tokens=1 << 17, cu=16, max_q=1 << 17, max_k=1 << 17, width=1 << 13) == 0
    with pytest.raises(AssertionError, match="null"):
        _lib.call("dcp_paged_attn", None, 0, 0, 0)


def test_the_arguments_have_the_size_the_library_takes(tmp_path):
    (tmp_path / "size.cpp").write_text('#include <stddef.h>\n#include "dcp_hip.h"\nstatic_assert(sizeof(dcp_paged_attn_args) == %d, "");\n'
                                       'static_assert(offsetof(dcp_paged_attn_args, softmax_scale) == %d, "");\n' % (_PAGED_ARGS.size, _PAGED_ARGS.size - 8))
    subprocess.run(["g++", "-fsyntax-only", f"-I{Path(__file__).resolve().parents[1] / 'include'}", str(tmp_path / "size.cpp")], check=True)
