"""gather_tokens over tables whose entries are no pages."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_append_tokens_gpu import DEV, make_cache

pytestmark = pytest.mark.gpu
BF16, F32, E4M3, INT8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("pool", [BF16, F32, E4M3, INT8])
@pytest.mark.parametrize("entry", [-1, -3, 10**6])
@pytest.mark.parametrize("d", [64, 12, 7])
def test_tokens_without_a_page_are_zeros(pool, entry, d):
    """They are not read from another sequence's page, and a notice is left."""
    cache = make_cache(pool, [100, 40], 0, 2, d, 16)
    want = ax.gather_tokens(cache, None, 100, dtype=F32)
    cache.block_table[0, 2] = entry  # tokens 32 .. 47
    cache.block_table[1, 3:] = entry  # (none)
    _lib.device_status()
    got = ax.gather_tokens(cache, None, 100, dtype=F32)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    for x, y in zip(got, want):
        assert bool((x[0, :, 32:48] == 0).all())
        y[0, :, 32:48] = 0
        assert torch.equal(x, y)
    ax.gather_tokens(cache, torch.tensor([48, 0], device=DEV), 50)
    assert _lib.device_status() == 0
