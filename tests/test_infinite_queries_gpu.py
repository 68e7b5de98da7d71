"""8-bit attention of query rows that hold infinities."""

import math

import pytest
import torch

import attnax_b200 as ax
from tests.test_append_tokens_gpu import DEV, as_bytes, make_cache
from tests.test_quantized_gpu import query

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("hq,t", [(2, 1), (4, 5), (4, 30)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_rows_with_one_sign_of_infinity(dt, pool, hq, t, sign):
    """Scores that are all -inf are no row without keys: its softmax is NaN, as with +inf.  Rows that see no key stay
    zeros, other rows as they were."""
    cache = make_cache(pool, [300, 3], 0, 1, 64, 16)
    cache.key_pool.copy_(torch.ones(cache.key_pool.shape, device=DEV).to(pool))
    q = query(cache, hq, t, dt)
    want = ax.paged_quantized_attention(q, cache)
    assert not bool(torch.isnan(want).any())
    q[:, 1, :, 7] = sign * math.inf
    q[:, 0, 0, 3] = sign * math.inf
    got = ax.paged_quantized_attention(q, cache)
    bad = torch.zeros(2, hq, t, dtype=torch.bool, device=DEV)
    bad[:, 1], bad[:, 0, 0] = True, True
    sees = torch.tensor([300, 3], device=DEV)[:, None] - t + torch.arange(t, device=DEV) >= 0
    bad &= sees[:, None]
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])
