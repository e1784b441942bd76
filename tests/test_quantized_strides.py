"""Keys and values at strides of their own: what the entry points of a cache in 4 bits take and refuse (CPU: nothing is launched)."""

import pytest
import torch

from dcp_amd import _lib
from dcp_amd.ops import quantized_cache_read, quantized_cache_write
from tests.test_quantized_refusals import _empty, built, here  # noqa: F401

ROWS = dict(n_tokens=3, heads=2, head_dim=64, dtype=0, k_token=128, k_head=64, v_token=640, v_head=64, n_pages=4, page_size=16, page=2176,
            cache_head=1088, stream=0)
CALLS = {"dcp_quantized_cache_write_strided": dict(k=16, v=16, slots=16, cache=16, **ROWS),
         "dcp_quantized_cache_read_strided": dict(cache=16, slots=16, k=16, v=16, **ROWS)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("wrong,message", [
    (dict(k_token=-128), "multiples of 8"), (dict(k_head=4), "multiples of 8"), (dict(v_token=-640), "multiples of 8"), (dict(v_head=68), "multiples of 8"),
    (dict(v_token=12), "multiples of 8"), (dict(page=8), "multiples of 16"), (dict(k=24), "aligned"), (dict(v=18), "aligned"), (dict(v=0), "null"),
    (dict(n_tokens=2**31 - 1, heads=1 << 12), "too many rows"), (dict(dtype=2), "bf16 and fp16"), (dict(head_dim=96), "head_dim")])
def test_refused(name, wrong, message):
    with pytest.raises(ValueError if message in ("bf16 and fp16", "head_dim") else AssertionError, match=message):
        _lib.call(name, *{**CALLS[name], **wrong}.values())


@pytest.mark.parametrize("name", CALLS)
def test_strides_of_an_axis_of_one_are_not_looked_at(name):
    odd = dict(k_token=3, v_token=-5)
    with pytest.raises(AssertionError, match="multiples of 8"):
        _lib.call(name, *{**CALLS[name], **odd}.values())
    with pytest.raises(AssertionError, match="null"):  # (what is asked next)
        _lib.call(name, *{**CALLS[name], **odd, "n_tokens": 1, "slots": 0}.values())
    with pytest.raises(AssertionError, match="null"):
        _lib.call(name, *{**CALLS[name], "k_head": 1, "v_head": -1, "heads": 1, "slots": 0}.values())


def test_strides_that_differ_are_passed_on(here):  # noqa: F811
    k, v = _empty(3, 2, 64), _empty(3, 10, 64)[:, 4:6]  # freshly made, and a slice of a fused projection
    slots, cache = _empty(3, dtype=torch.int64), _empty(4, 2, 1, 17 * 64, dtype=torch.uint8)
    quantized_cache_write(k, v, slots, cache)
    quantized_cache_read(cache, slots, out=(v, k))
    quantized_cache_write(k[:1], v[:1], slots[:1], cache)  # (the strides of one token say nothing, but they differ)
    quantized_cache_write(k, k, slots, cache)
    assert [(call[0], call[9:13]) for call in here[:3]] == [("dcp_quantized_cache_write_strided", (128, 64, 640, 64)),
                                                            ("dcp_quantized_cache_read_strided", (640, 64, 128, 64)),
                                                            ("dcp_quantized_cache_write_strided", (128, 64, 640, 64))]
    assert here[3][0] == "dcp_quantized_cache_write" and here[3][9:11] == (128, 64)


@pytest.mark.parametrize("wrong", ["heads", "tokens", "dim", "rows", "type", "slots", "v_slots"])
def test_rows_that_do_not_belong_together(here, wrong):  # noqa: F811
    k, v, slots, cache = _empty(3, 2, 64), _empty(3, 10, 64)[:, 4:6], _empty(3, dtype=torch.int64), _empty(4, 2, 1, 17 * 64, dtype=torch.uint8)
    args = dict(heads=(k, _empty(3, 10, 64)[:, 4:7], slots), tokens=(k, v[:2], slots), dim=(k, _empty(3, 10, 128)[:, 4:6], slots),
                rows=(k, _empty(3, 2, 128)[..., ::2], slots), type=(k, _empty(3, 10, 64, dtype=torch.float16)[:, 4:6], slots),
                slots=(k, v, slots.int()), v_slots=(k, v, _empty(4, dtype=torch.int64)))[wrong]
    for call in (lambda: quantized_cache_write(*args, cache), lambda: quantized_cache_read(cache, args[2], out=args[:2])):
        with pytest.raises((ValueError, TypeError)):
            call()
    assert not here
