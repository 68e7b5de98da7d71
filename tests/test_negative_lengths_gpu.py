"""A sequence whose length is negative gets no tokens, in either kind of pool."""

import dataclasses

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_append_tokens_gpu import DEV, as_bytes, make_cache, snapshot

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool", [torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("length,t", [(-2, 5), (-1, 1), (-1, 40), (-2**31, 3), (-20, 20)])
def test_nothing_is_written(pool, length, t):
    cache = make_cache(pool, [20, 40, 5], t)
    cache = dataclasses.replace(cache, seq_lengths=torch.tensor([20, length, 5], dtype=torch.int32, device=DEV))
    k, v = (torch.randn(3, 2, t, 64, device=DEV) for _ in range(2))
    before = snapshot(cache)
    with pytest.raises(ValueError, match="sequence 1"):
        ax.append_tokens(cache, k, v)
    _lib.device_status()
    out = ax.append_tokens(cache, k, v, check=False)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    assert out.seq_lengths.tolist() == [20 + t, length + t, 5 + t]
    mine = cache.block_table[1][cache.block_table[1] >= 0].long()
    for name in ("key_pool", "value_pool", "key_scales", "value_scales"):
        if name in before:
            assert torch.equal(as_bytes(getattr(out, name))[mine], as_bytes(before[name])[mine])
    want = ax.append_tokens(dataclasses.replace(cache, seq_lengths=before["seq_lengths"], **{
        name: x.clone() for name, x in before.items() if "pool" in name or "scales" in name}), k, v,
        new_lengths=[t, 0, t], check=False)
    assert _lib.device_status() == 0
    for name in ("key_pool", "value_pool"):  # the other sequences are complete
        assert torch.equal(as_bytes(getattr(out, name)), as_bytes(getattr(want, name)))
