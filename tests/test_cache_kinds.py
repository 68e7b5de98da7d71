"""Caches that only have the four fields of a paged cache go through the page operators (host side; no GPU)."""

import typing

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib, pages


class Four(typing.NamedTuple):
    key_pool: torch.Tensor
    value_pool: torch.Tensor
    block_table: torch.Tensor
    seq_lengths: torch.Tensor

    num_blocks = property(lambda self: int(self.key_pool.shape[0]))
    block_size = property(lambda self: int(self.key_pool.shape[1]))
    num_kv_heads = property(lambda self: int(self.key_pool.shape[2]))
    head_dim = property(lambda self: int(self.key_pool.shape[3]))


class Sub(ax.PagedKVCache):
    """A program's own kind of cache."""


def four(kind, **kw):
    pool = torch.zeros(8, 16, 2, 8, dtype=torch.bfloat16, **kw)
    return kind(pool, torch.zeros_like(pool), torch.full((2, 3), -1, dtype=torch.int32, **kw),
                torch.zeros(2, dtype=torch.int32, **kw))


@pytest.mark.parametrize("kind", [Four, Sub, ax.PagedKVCache])
def test_allocate_blocks(kind):
    cache, n = ax.allocate_blocks(four(kind), sequence_idx=1, num_new_tokens=20, free_block_ids=[5, 3, 1])
    assert n == 2 and type(cache) is ax.PagedKVCache and cache.block_table.tolist() == [[-1] * 3, [5, 3, -1]]


@pytest.mark.parametrize("kind", [Four, Sub, ax.PagedKVCache])
def test_results_of_page_operators(monkeypatch, kind):
    """The launches left out: what counts is what comes back."""
    monkeypatch.setattr(_lib, "run", lambda *a: None)
    params = pages._params

    def on_host(cache):  # (the check that the pools are on the GPU is all that is left out)
        monkeypatch.setattr(torch.Tensor, "is_cuda", True)
        try:
            return params(cache)
        finally:
            monkeypatch.undo()
            monkeypatch.setattr(_lib, "run", lambda *a: None)
            monkeypatch.setattr(pages, "_params", on_host)

    monkeypatch.setattr(pages, "_params", on_host)
    c = four(kind)
    for out in (ax.fork_sequences(c, [0], [1], [2])[0], ax.free_sequences(c, [0])[0],
                ax.free_window(c, window_size=4)[0], ax.compact_blocks(c)[0]):
        assert type(out) is ax.PagedKVCache and out.key_pool is c.key_pool and out.value_pool is c.value_pool


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [Four, Sub])
def test_on_the_gpu(kind):
    free = [5, 3, 1, 0]
    a, b = four(kind, device="cuda"), four(ax.PagedKVCache, device="cuda")
    x = torch.randn(2, 2, 4, 8, device="cuda").to(torch.bfloat16)
    for c in (a, b):
        c.block_table[0, :2] = torch.tensor([6, 4], dtype=torch.int32)
        c.seq_lengths[0] = 18
    idx, n = torch.tensor([[0, 2], [0, 0]], dtype=torch.int32), torch.tensor([2, 0], dtype=torch.int32)
    a, b = (ax.append_accepted(c, x, x, idx, n) for c in (a, b))
    a, b = (ax.fork_sequences(c, [0], [1], free)[0] for c in (a, b))
    a, b = (ax.free_window(c, window_size=3)[0] for c in (a, b))
    a, b = (ax.compact_blocks(c)[0] for c in (a, b))
    for name in Four._fields:
        assert torch.equal(getattr(a, name), getattr(b, name))
    assert a.seq_lengths.tolist() == [20, 20]


def test_codes_are_refused_by_append_accepted():
    q = ax.init_quantized_paged_kv_cache(num_blocks=4, block_size=16, num_kv_heads=2, head_dim=8, batch_size=2,
                                         max_blocks_per_seq=2, device="cpu")
    x = torch.zeros(2, 2, 3, 8)
    with pytest.raises(ValueError, match="append_tokens"):
        ax.append_accepted(q, x, x, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
