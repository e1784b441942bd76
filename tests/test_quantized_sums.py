"""Calls over a cache in 4 bits with so many units that 32 bits do not hold what the kernel of few rows adds up (CPU: nothing is launched)."""

import pytest

from dcp_amd import _lib
from dcp_amd.flash_attn_interface import _QUANTIZED_ARGS
from tests.test_quantized_refusals import ATTN, built  # noqa: F401

# one key each, but said to be long: units of one turn and three for their start, 2^31 in all
MANY = {**ATTN, **dict(n_tokens=1 << 16, batch=1 << 16, heads=1 << 13, kv_heads=1 << 13, head_dim=64, width=1, max_q=1, max_k=1 << 20)}


def _workspace(**changed):
    return _lib.load().dcp_quantized_attn_workspace_bytes(_QUANTIZED_ARGS.pack(*{**MANY, **changed}.values()))


def test_the_kernel_of_few_rows_has_no_more_than_it_can_count():
    """It says where every row's pieces are, 8 bytes a row, the kernel of rows nothing where it takes a row's keys at once."""
    rows = MANY["n_tokens"] * MANY["heads"]
    assert _workspace() == 0
    assert _workspace(n_tokens=1 << 14, batch=1 << 14) >= 8 * rows / 4


def test_more_work_items_than_a_launch_can_have():
    with pytest.raises(AssertionError, match="too many work items"):
        _lib.call("dcp_quantized_attn", _QUANTIZED_ARGS.pack(*MANY.values()), 16, 1 << 40, 0)
