"""8-bit attention: the shares of warps and splits are joined without passing either end of fp32."""

import math

import pytest
import torch

import attnax_b200 as ax
from tests.test_append_tokens_gpu import DEV, make_cache
from tests.test_quantized_gpu import attention64, check

pytestmark = pytest.mark.gpu
BF16, F32, E4M3, INT8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8
ROWS = [(1, 1), (4, 1), (8, 3), (4, 8), (8, 10)]  # query heads over one kv head, T


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("hq,t", ROWS)
@pytest.mark.parametrize("lens", [40, 700, 9000])
def test_means_of_the_largest_values(pool, lens, hq, t):
    """Sums of these values pass fp32, their means do not."""
    cache = make_cache(pool, [lens], 0, 1, 64, 16, seed=lens)
    cache.value_scales.fill_(2.0 ** 119)
    cache.value_pool.copy_(torch.full(cache.value_pool.shape, 240.0 if pool == E4M3 else 127.0, device=DEV).to(pool))
    q = torch.randn(1, hq, t, 64, device=DEV) * 0.5
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("hq,t", ROWS)
@pytest.mark.parametrize("below,large", [(90.0, 2.0 ** 20), (126.0, 2.0 ** 30), (138.0, 2.0 ** 30), (230.0, 2.0 ** 119)])
def test_weights_that_fp32_does_not_hold(pool, hq, t, below, large):
    """The second block's scores lie ``below`` (log2) under the first one's, whose values are tiny: what it adds counts
    all the same.  Few rows: page by page in another warp; many: in another split.  Both: far apart, in another split."""
    for first, rest in ([(128, 128), (512, 512)] if hq * t >= 49 else [(16, 16), (512, 512)]):
        cache = make_cache(pool, [first + rest], 0, 1, 64, 16, seed=first)
        table = cache.block_table[0].long()
        back = table[first // 16:]
        keys = torch.ones(cache.key_pool.shape, device=DEV)
        keys[back] = -1.0
        cache.key_pool.copy_(keys.to(pool))
        cache.key_scales.fill_(2.0)
        cache.value_scales.fill_(2.0 ** -100)
        cache.value_scales[back] = large
        if large > 2.0 ** 110:  # (codes up to 120: what they stand for stays finite)
            cache.value_pool[back] = torch.ones((), device=DEV).to(pool)
        x = below * math.log(2.0) / (2 * 2.0 * 8)  # scores of +-2 x sqrt(64)
        q = torch.full((1, hq, t, 64), x, device=DEV, dtype=F32)
        check(ax.paged_quantized_attention(q, cache), attention64(q, cache))
