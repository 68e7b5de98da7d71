"""8-bit attention of long chunks of prompts, with and without a prefix, some padded in front."""

import pytest
import torch

import attnax_b200 as ax
from tests.test_append_tokens_gpu import DEV, make_cache
from tests.test_quantized_gpu import attention64, check, query

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("pool,dt", [(E4M3, BF16), (INT8, F16), (E4M3, F32)])
@pytest.mark.parametrize("lens,t,hq,hk,d,bs", [
    ([512, 700], 512, 2, 1, 128, 16),     # one prompt without a prefix
    ([1001, 3000, 40, 0], 1001, 1, 1, 64, 32),
    ([2300], 777, 6, 2, 64, 64),
    ([600, 129], 600, 5, 5, 128, 48),
])
def test_against_64_bits(pool, dt, lens, t, hq, hk, d, bs):
    cache = make_cache(pool, lens, 0, hk, d, bs, seed=t)
    q = query(cache, hq, t, dt)
    want = attention64(q, cache)
    check(ax.paged_quantized_attention(q, cache), want, "lengths read")
    check(ax.paged_quantized_attention(q, cache, max_context=max(lens) + 900), want, "bounded")


def test_a_prompt_in_chunks_equals_its_rows_at_once():
    """Appended and attended chunk by chunk, or all at once: scales of a page may grow in between, so pages are filled
    chunk by chunk first and read at both widths."""
    cache = make_cache(E4M3, [1500], 0, 2, 64, 16)
    q = query(cache, 8, 1500)
    want = attention64(q, cache)
    check(ax.paged_quantized_attention(q, cache), want)
    for first, last in ((0, 100), (100, 612), (612, 1500)):
        part = ax.QuantizedPagedKVCache(cache.key_pool, cache.value_pool, cache.key_scales, cache.value_scales,
                                        cache.block_table, torch.full_like(cache.seq_lengths, last))
        check(ax.paged_quantized_attention(q[:, :, first:last], part), tuple(x[:, :, first:last] for x in want))
