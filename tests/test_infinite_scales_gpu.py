"""8-bit attention beside a page whose value scale is infinite."""

import math

import pytest
import torch

import attnax_b200 as ax
from tests.test_append_tokens_gpu import make_cache
from tests.test_quantized_gpu import query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("hq", [2, 4, 32])
def test_only_rows_that_see_the_page_are_touched(pool, hq):
    cache = make_cache(pool, [40], 0, 2, 64, 16)
    q = query(cache, hq, 12)  # rows at 28 .. 39
    want = ax.paged_quantized_attention(q, cache)
    cache.value_scales[int(cache.block_table[0, 2])] = math.inf  # tokens 32 .. 39
    got = ax.paged_quantized_attention(q, cache)
    assert not bool(torch.isfinite(got[:, :, 4:]).any())
    assert torch.equal(got[:, :, :4], want[:, :, :4])
