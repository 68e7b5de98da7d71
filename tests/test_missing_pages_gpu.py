"""8-bit attention and reads over tables whose entries are no pages: freed ones, or out of range."""

import dataclasses

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_append_tokens_gpu import DEV, as_bytes, make_cache, snapshot
from tests.test_quantized_gpu import attention64, check, query

pytestmark = pytest.mark.gpu
BF16, F32, E4M3, INT8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8
LENS = [300, 40, 700]


def expected(q, cache):
    """Caches off the fused kernel's shapes run the window kernels on bf16, which round P to bf16: half a step is 2^-8
    of a weight there, where the fused kernel's fp16 has 2^-11."""
    return attention64(q, cache, sixteen=cache.block_size % 16 != 0 or cache.head_dim not in (64, 128))


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("hq,t", [(4, 1), (4, 12), (4, 40)])
@pytest.mark.parametrize("bs,d", [(16, 64), (48, 128), (24, 64), (8, 32), (16, 80)])
@pytest.mark.parametrize("bounded", [False, True])
def test_rows_without_a_page_are_nan(pool, hq, t, bs, d, bounded):
    """Pages taken by free_window are not read as the pool's last one: rows that stand behind them are NaN."""
    cache = make_cache(pool, LENS, 0, 2, d, bs, seed=t)
    q = query(cache, hq, t)
    want = expected(q, cache)
    freed, _, count = ax.free_window(cache, window_size=200)
    assert int(count) > 0 and bool((freed.block_table[1] == cache.block_table[1]).all())
    _lib.device_status()
    if d == 80:  # (a head dim that the flash kernels do not have is refused)
        with pytest.raises(NotImplementedError):
            ax.paged_quantized_attention(q, freed, max_context=max(LENS) if bounded else None)
        _lib.device_status()
        return
    got = ax.paged_quantized_attention(q, freed, max_context=max(LENS) if bounded else None)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[2]).all())
    check(got[1:2], tuple(x[1:2] for x in want))
    check(ax.paged_quantized_attention(q, cache), want)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("entry", [-1, -7, 10**6])
@pytest.mark.parametrize("bs", [16, 24])
@pytest.mark.parametrize("t", [12, 60])
def test_rows_in_front_of_the_missing_page_are_not_touched(entry, bs, t):
    cache = make_cache(E4M3, [100], 0, 2, 64, bs)
    q = query(cache, 4, t)
    want = expected(q, cache)
    last = cache.block_table.shape[1] - 1  # tokens from last * bs on
    bad = dataclasses.replace(cache, block_table=cache.block_table.clone())
    bad.block_table[0, last] = entry
    _lib.device_status()
    got = ax.paged_quantized_attention(q, bad)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    sees = 100 - t + torch.arange(t, device=DEV) >= last * bs
    assert bool(torch.isnan(got[:, :, sees]).all()) and bool(sees.any()) and not bool(sees.all())
    check(got[:, :, ~sees], tuple(x[:, :, ~sees] for x in want))


def test_nothing_visible_nothing_noted():
    """Entries behind the sequence, and those of empty sequences, are not looked at."""
    cache = make_cache(INT8, [40, 0], 0, 2, 64, 16)
    cache.block_table[1] = -1
    cache.block_table[0, 3:] = -1
    _lib.device_status()
    for t in (1, 40):
        q = query(cache, 4, t)
        check(ax.paged_quantized_attention(q, cache), expected(q, cache))
    assert _lib.device_status() == 0
