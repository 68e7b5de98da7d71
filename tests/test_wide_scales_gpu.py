"""8-bit attention over pages whose value scales lie many powers of two apart, and over values near fp32's largest."""

import math

import pytest
import torch

import attnax_b200 as ax
from tests.test_append_tokens_gpu import DEV, as_bytes, make_cache
from tests.test_quantized_gpu import attention64, check

pytestmark = pytest.mark.gpu
BF16, F32, E4M3, INT8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8

# Tokens 0 .. 15 have the largest scores; how far (log2) those of the last page lie below them is `below`.
ROWS = [(1, 1), (4, 1), (8, 3), (4, 8), (8, 10)]  # query heads over one kv head, T


def two_levels(pool, lens, below, small, large, d=64):
    """Pages of value scale ``small`` and the largest scores, the last one with ``large`` and scores ``below`` less.

    Keys are +1 or -1 in every channel, queries alike: a score is +-x d / sqrt(d).
    """
    cache = make_cache(pool, [lens], 0, 1, d, 16, seed=lens)
    table = cache.block_table[0].long()
    keys = torch.ones(cache.key_pool.shape, device=DEV)
    keys[table[-1]] = -1.0
    cache.key_pool.copy_(keys.to(pool))
    cache.key_scales.fill_(2.0)
    cache.value_scales.fill_(small)
    cache.value_scales[table[-1]] = large
    x = below * math.log(2.0) / (2 * 2.0 * math.sqrt(d))  # scores of +-2 x sqrt(d)
    return cache, table, x


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("lens,below,large", [
    # one tile of 128 tokens and one warp's units (64 tokens apart); the factor 2^(log2 scale + maxima apart) passes
    # fp32, and the far page's share runs from the largest contribution to nothing
    (80, 118.0, 2.0 ** 20), (80, 126.0, 2.0 ** 30), (80, 138.0, 2.0 ** 30), (80, 150.0, 2.0 ** 60), (80, 230.0, 2.0 ** 119),
    (80, 215.0, 2.0 ** 119), (400, 130.0, 2.0 ** 30), (336, 90.0, 2.0 ** 20),
])
@pytest.mark.parametrize("hq,t", ROWS)
def test_small_scales_with_the_large_weights(pool, zeros, lens, below, large, hq, t):
    cache, table, x = two_levels(pool, lens, below, 2.0 ** -100, large)
    if zeros:
        as_bytes(cache.value_pool)[table[:-1]] = 0
    if large > 2.0 ** 110:  # (codes up to 120: what they stand for stays finite)
        as_bytes(cache.value_pool)[table[-1]] = as_bytes(torch.ones((), device=DEV).to(pool))
    q = torch.full((1, hq, t, 64), x, device=DEV, dtype=F32)
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))
    q = q.to(BF16)
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))
