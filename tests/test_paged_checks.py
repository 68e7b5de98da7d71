"""What the paged entry points refuse about the cache itself, without a GPU: its fields have to describe each other."""

import pytest
import torch

import attnax_b200 as ax

BF = torch.bfloat16


def cpu_cache():
    return ax.init_paged_kv_cache(num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, batch_size=3,
                                  max_blocks_per_seq=4, device="cpu")


Q = torch.zeros(3, 4, 2, 64, dtype=BF)
DRAFT = torch.zeros(3, 2, 2, 64, dtype=BF)
PAR = torch.full((3, 2), -1, dtype=torch.int32)

ROWS = [
    lambda c: ax.paged_window_attention(Q, c, window_size=4),
    lambda c: ax.paged_tree_attention(Q, DRAFT, DRAFT, c, PAR),
]
PAGES = [
    lambda c: ax.copy_blocks(c, [0], [1]), lambda c: ax.fork_sequences(c, [0], [1], [2]),
    lambda c: ax.free_sequences(c, [0]), lambda c: ax.free_window(c, window_size=3),
    lambda c: ax.compact_blocks(c), lambda c: ax.append_accepted(c, DRAFT, DRAFT, [[0]] * 3, [1] * 3),
]
OLDER = [
    lambda c: ax.append_kv(c, 0, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64)),
    lambda c: ax.gather_kv(c, 0),
    lambda c: ax.paged_attention_batched(torch.zeros(3, 4, 2, 64, dtype=BF), c),
]

POOLS = {
    "fewer pages": lambda v: v[:4], "smaller pages": lambda v: v[:, :8], "fewer heads": lambda v: v[:, :, :1],
    "smaller head": lambda v: v[..., :32], "wider": lambda v: v.float(), "other type": lambda v: v.to(torch.float16),
    "flat": lambda v: v.flatten(),
}


@pytest.mark.parametrize("call", ROWS + PAGES + OLDER)
@pytest.mark.parametrize("pool", POOLS)
def test_value_pool_unlike_the_key_pool(call, pool):
    c = cpu_cache()
    with pytest.raises(ValueError, match="value_pool"):
        call(ax.PagedKVCache(c.key_pool, POOLS[pool](c.value_pool), c.block_table, c.seq_lengths))


@pytest.mark.parametrize("call", ROWS + PAGES + OLDER)
def test_value_pool_on_another_device(call):
    c = cpu_cache()
    with pytest.raises(RuntimeError, match="value_pool"):
        call(ax.PagedKVCache(c.key_pool, c.value_pool.to("meta"), c.block_table, c.seq_lengths))


@pytest.mark.parametrize("call", ROWS + PAGES)
def test_lengths_and_table_rows_that_do_not_match(call):
    c = cpu_cache()
    for table, lens in ((c.block_table, c.seq_lengths[:2]), (c.block_table, c.seq_lengths[None]),
                        (c.block_table, c.seq_lengths[0]), (c.block_table.flatten(), c.seq_lengths),
                        (c.block_table[None], c.seq_lengths), (c.block_table, torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(ax.PagedKVCache(c.key_pool, c.value_pool, table, lens))


def test_decode_rows():
    from attnax_b200.paged import paged_decode_raw

    c = cpu_cache()
    for q, kw in ((Q[:2], {}), (torch.cat([Q, Q]), {}), (Q, {"seq_lengths": c.seq_lengths[:2]}),
                  (Q, {"block_table": c.block_table[:2]}), (Q, {"block_table": c.block_table[0]})):
        with pytest.raises(ValueError):
            paged_decode_raw(q, c, **kw)


def test_wide_integers_are_not_cut_to_their_low_half():
    from attnax_b200.paged_rows import on_device

    dev = torch.device("cpu")
    far = [1 << 32, -(1 << 32), (1 << 40) + 5, 7, -1, 2**31 - 1, -2**31]
    want = [2**31 - 1, -2**31, 2**31 - 1, 7, -1, 2**31 - 1, -2**31]
    for x in (far, torch.tensor(far)):
        got = on_device(x, dev)
        assert got.dtype == torch.int32 and got.tolist() == want
    assert on_device(torch.tensor([3, 250], dtype=torch.uint8), dev).tolist() == [3, 250]
    assert on_device([], dev).tolist() == []


@pytest.mark.parametrize("wrong", [torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.bool)])
def test_indices_must_be_integers(wrong):
    c = cpu_cache()
    with pytest.raises(ValueError):
        ax.paged_tree_attention(Q, DRAFT, DRAFT, c, wrong)
    with pytest.raises(ValueError):
        ax.paged_tree_attention(Q, DRAFT, DRAFT, c, PAR, tree_lengths=wrong[:, 0])
    with pytest.raises(ValueError):
        ax.append_accepted(c, DRAFT, DRAFT, wrong, [1] * 3)
    with pytest.raises(ValueError):
        ax.append_accepted(c, DRAFT, DRAFT, [[0]] * 3, wrong[:, 0])


@pytest.mark.parametrize("call", ROWS + PAGES + OLDER)
def test_tables_and_lengths_of_other_types(call):
    c = cpu_cache()
    for table, lens in ((c.block_table.long(), c.seq_lengths), (c.block_table, c.seq_lengths.long()),
                        (c.block_table.to(torch.int16), c.seq_lengths), (c.block_table, c.seq_lengths.float())):
        with pytest.raises(ValueError, match="int32"):
            call(ax.PagedKVCache(c.key_pool, c.value_pool, table, lens))
