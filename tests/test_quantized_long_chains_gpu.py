"""Prompts over a cache in 4 bits whose workgroups go through more tiles than the table of their places holds at once: 64-key tiles, 2 x 64 of
them, a half looked up again while the other is used."""

import pytest
import torch

from dcp_amd.flash_attn_interface import quantized_cache_attention
from tests.paged_cases import check
from tests.quantized_cases import Quantized

pytestmark = pytest.mark.gpu
F16 = torch.float16
# around where a half is looked up (32 and 96 tiles behind a multiple of 128) and where it is used for the first time
EDGES = (31, 32, 33, 63, 64, 66, 95, 96, 97, 99, 127, 128, 130, 160, 191, 192, 223, 224, 225, 255, 256)


def _whole(gpu, case):
    """Not cut: as far as the host knows there is one key."""
    got = quantized_cache_attention(**{**case.to(gpu), "max_seqlen_k": 1})
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("more", [dict(), dict(head_dim=64, dtype=F16), dict(window=9000, n_starting=100), dict(window=9000, n_starting=100, head_dim=64)])
@pytest.mark.parametrize("new", [50, 20])
def test_more_tiles_than_the_table_holds(gpu, new, more):
    case = Quantized([17500], new=[new], heads=2, kv_heads=1, **more)
    check(_whole(gpu, case), case.truth())


@pytest.mark.parametrize("beside", [0, 64])
def test_chains_that_end_at_the_edges(gpu, beside):
    """And of so many requests that they are not ranked by their lengths."""
    keys = [6080, 6144, 6145, 8128, 8192, 8193, 10240, 10300]
    case = Quantized(keys + [5] * beside, new=[40] * len(keys) + [1] * beside, heads=2, kv_heads=1, head_dim=64)
    check(_whole(gpu, case), case.truth())


@pytest.mark.parametrize("window", [0, 13000])
@pytest.mark.parametrize("new", [50, 20])
def test_missing_pages_at_the_edges(gpu, new, window):
    """The first, the last or an inner 16 keys of the tiles there are of no page."""
    n, n_starting = 17500, 100 if window else 0
    n_first, begin = (-(-n_starting // 16), (n - new - window + 1) // 16) if window else (0, 0)
    groups = [4 * tile + i % 4 for i, tile in enumerate(EDGES)]
    pages = [g if g < n_first else g - n_first + begin for g in groups]
    case = Quantized([n], new=[new], bad=[(0, page, lambda n: -1) for page in pages if page < -(-n // 16)], page_size=16, heads=2, kv_heads=1,
                     head_dim=64, window=window, n_starting=n_starting)
    assert (case.table < 0).sum() == (16 if window else 21)  # (of a window's tiles there are 206)
    check(_whole(gpu, case), case.truth())
