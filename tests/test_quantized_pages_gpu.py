"""The page operators on 8-bit caches: scales go with their pages.  Each is held to the same call on an fp32 cache of
the values that the codes stand for."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_append_tokens_gpu import BITS8, DEV, as_bytes, make_cache

pytestmark = pytest.mark.gpu


def values(cache):
    return tuple(p.float() * s[:, None, :, None] for p, s in ((cache.key_pool, cache.key_scales),
                                                              (cache.value_pool, cache.value_scales)))


def pair(pool, lens, hk=2, d=64, bs=16, spare=9, seed=0, room=0):
    q = make_cache(pool, lens, room, hk, d, bs, seed, spare)
    return q, ax.PagedKVCache(*values(q), q.block_table.clone(), q.seq_lengths.clone())


def same(q, wide):
    assert isinstance(q, ax.QuantizedPagedKVCache) and isinstance(wide, ax.PagedKVCache)
    assert torch.equal(q.block_table, wide.block_table) and torch.equal(q.seq_lengths, wide.seq_lengths)
    k, v = values(q)
    assert torch.equal(k, wide.key_pool) and torch.equal(v, wide.value_pool)


SHAPES = [(2, 64, 16), (8, 128, 32), (1, 3, 5), (3, 7, 1), (1, 10, 3)]


@pytest.mark.parametrize("pool", BITS8)
@pytest.mark.parametrize("hk,d,bs", SHAPES)
@pytest.mark.parametrize("device", ["cpu", DEV])
def test_copy(pool, hk, d, bs, device):
    q, wide = pair(pool, [60], hk, d, bs, spare=60)
    perm = torch.randperm(q.num_blocks, generator=torch.Generator().manual_seed(3))
    src, dst = perm[:25].to(torch.int32).to(device), perm[25:50].to(torch.int32).to(device)
    same(ax.copy_blocks(q, src, dst), ax.copy_blocks(wide, src, dst))


@pytest.mark.parametrize("pool", BITS8)
def test_copy_many_pages(pool):
    q, wide = pair(pool, [1], 2, 16, 4, spare=3000)
    perm = torch.randperm(q.num_blocks, generator=torch.Generator().manual_seed(4)).to(torch.int32).to(DEV)
    same(ax.copy_blocks(q, perm[:1300], perm[1300:2600]), ax.copy_blocks(wide, perm[:1300], perm[1300:2600]))


@pytest.mark.parametrize("pool", BITS8)
@pytest.mark.parametrize("hk,d,bs", SHAPES)
def test_fork_append_and_free(pool, hk, d, bs):
    """A prompt is forked; both go on on their own pages; then rows end, and the pool is compacted."""
    q, wide = pair(pool, [0, 37, 0, 2 * bs], hk, d, bs, spare=12)
    held = set(q.block_table[q.block_table >= 0].tolist())
    free = [i for i in range(q.num_blocks) if i not in held]
    (q2, used), (w2, want) = (ax.fork_sequences(c, [1, 3], [0, 2], free[:2]) for c in (q, wide))
    assert int(used) == int(want)
    same(q2, w2)
    if 37 % bs:  # the fork's open page is its own: what it appends does not show in its source
        k0, _ = ax.gather_tokens(q2, None, 37, dtype=torch.float32)
        x = torch.full((4, hk, 1, d), 7.0, device=DEV)
        q3 = ax.append_tokens(q2, x, x, new_lengths=[1, 0, 0, 0])
        k1, _ = ax.gather_tokens(q3, None, 38, dtype=torch.float32)
        assert torch.equal(k1[1, :, :37], k0[1]) and bool((k1[0, :, 37] == 7).all())
        w2 = ax.PagedKVCache(*values(q3), q3.block_table, q3.seq_lengths)
        q2 = q3
    (q4, freed, n), (w4, freed_w, n_w) = (ax.free_sequences(c, [1]) for c in (q2, w2))
    assert torch.equal(freed, freed_w) and int(n) == int(n_w)
    same(q4, w4)
    (q5, live), (w5, live_w) = (ax.compact_blocks(c) for c in (q4, w4))
    assert int(live) == int(live_w)
    same(q5, w5)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("pool", BITS8)
def test_free_window(pool):
    q, wide = pair(pool, [100, 5, 0, 64])
    (a, f, n), (b, g, m) = (ax.free_window(c, window_size=20, num_sinks=4) for c in (q, wide))
    assert torch.equal(f, g) and int(n) == int(m) > 0
    same(a, b)


@pytest.mark.parametrize("pool", BITS8)
def test_what_takes_other_caches_only(pool):
    cache = make_cache(pool, [20, 33], 8)
    q = torch.zeros(2, 4, 1, 64, device=DEV, dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 1, 64, device=DEV, dtype=torch.bfloat16)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    before = as_bytes(cache.key_pool).clone()
    for call in (lambda: ax.paged_attention_batched(q, cache), lambda: ax.paged_attention(q[0], cache, 0),
                 lambda: ax.paged_window_attention(q, cache, window_size=8),
                 lambda: ax.paged_tree_attention(q, k, k, cache, torch.full((2, 1), -1)),
                 lambda: ax.append_accepted(cache, k, k, torch.zeros(2, 1), lens),
                 lambda: ax.append_kv(cache, 0, k[0].transpose(0, 1), k[0].transpose(0, 1)),
                 lambda: ax.gather_kv(cache, 0)):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(before, as_bytes(cache.key_pool))
