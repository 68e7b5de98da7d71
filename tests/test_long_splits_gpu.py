"""8-bit attention over splits longer than the pages and scales that a warp's lanes hold at a time.

Partials are kept within 1 GiB by splits of twice the length, which takes many sequences: these share their pages.
"""

import ctypes
import dataclasses

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_append_tokens_gpu import DEV, make_cache
from tests.test_quantized_gpu import attention64, check, query

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def workspace(n, hq, hk, t, most):
    p = _lib.PagedAttend8Params()
    p.dtype, p.pool_format, p.num_seqs, p.num_heads_q, p.num_heads_kv = _lib.ATTN_BF16, _lib.POOL_E4M3, n, hq, hk
    p.head_dim, p.seq_q, p.num_blocks, p.block_size, p.max_blocks_per_seq, p.max_context = 64, t, 300, 16, 300, most
    return _lib.load().attn_paged_attend8_workspace_size(ctypes.byref(p))


@pytest.mark.parametrize("pool,hq,hk,t,n", [(E4M3, 16, 2, 4, 22000), (INT8, 64, 8, 1, 22000), (INT8, 16, 2, 4, 40000)])
def test_refilled_batches(pool, hq, hk, t, n):
    most, page = 4500, 16
    one = workspace(n, hq, hk, t, most)
    if n == 22000:  # two splits, of 4096 tokens: 64 units a warp where 32 are held at a time
        assert 2 * n * hq * t * 65 * 4 <= one + 4096 and one <= 2**30 < 3 * n * hq * t * 65 * 4
    else:
        assert one == 0  # one split, of all tokens
    cache = make_cache(pool, [most], 0, hk, 64, page)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    pages = cache.block_table[0]
    table = pages[torch.randint(0, pages.numel(), (n, pages.numel()), generator=g, device=DEV)].contiguous()
    lens = torch.randint(1, 200, (n,), generator=g, device=DEV, dtype=torch.int32)
    sample = [0, 1, 12345, n - 2, n - 1]
    lens[sample] = torch.tensor([most, 4097, 2100, 4096, 4480], dtype=torch.int32, device=DEV)
    many = dataclasses.replace(cache, block_table=table, seq_lengths=lens)
    q = query(many, hq, t)
    got = ax.paged_quantized_attention(q, many, max_context=most)[sample]
    few = dataclasses.replace(cache, block_table=table[sample].contiguous(), seq_lengths=lens[sample])
    check(got, attention64(q[sample], few))
