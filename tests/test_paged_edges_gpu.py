"""Window, tree and page operators at the edge of their contract."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests._plain64 import assert_within, attention64
from tests.test_paged_rows_gpu import check_tree, check_window, history, make_cache, randn, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
NAN = float("nan")


# rows per kv head: 2, 20 (warp MMA); 48, 160, 320 (tcgen05).  Contexts in one split, in a cluster, in joined splits.
@pytest.mark.parametrize("t,hq,hkv", [(1, 4, 2), (5, 4, 1), (12, 8, 2), (40, 4, 1), (40, 8, 1)])
@pytest.mark.parametrize("n", [60, 900, 9000])
@pytest.mark.parametrize("where", ["query", "key"])
def test_nan_stays_nan(t, hq, hkv, n, where):
    """A row whose scores hold NaN is NaN, as in the formula; the other sequence's rows are untouched."""
    lens = [n, n]
    cache = make_cache(t + n, lens, hkv, 128, 16, BF)
    q, dk, dv = randn(1, 2, hq, t, 128), randn(2, 2, hkv, t, 128), randn(3, 2, hkv, t, 128)
    par = random_tree(4, 2, t)
    if where == "query":
        q[0, 1, -1, 3] = NAN
    else:  # the newest key of sequence 0, seen by its last row (window) and by every row (tree)
        cache.key_pool[cache.block_table[0, (n - 1) // 16].long(), (n - 1) % 16, :, 5] = NAN
    window = ax.paged_window_attention(q, cache, window_size=n, num_sinks=2)
    tree = ax.paged_tree_attention(q, dk, dv, cache, par)
    for got in (window, tree):
        bad = got.isnan().any(-1)
        assert bool((bad == got.isnan().all(-1)).all())
        assert not bool(bad[1].any())
    if where == "query":
        assert bool(window[0, 1, -1].isnan().all()) and int(window.isnan().any(-1).sum()) == 1
        assert bool(tree[0, 1, -1].isnan().all()) and int(tree.isnan().any(-1).sum()) == 1
    else:
        assert bool(window[0, :, -1].isnan().all()) and int(window.isnan().any(-1).sum()) == hq
        assert bool(tree[0].isnan().all())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_nan_stays_nan_in_32_bits(d, masked):
    """fp32 with sinks: a row with a NaN score is no row without keys (zeros, or the mean of V under a mask)."""
    s, hq, hkv = 200, 4, 2
    q, k, v, do = (randn(i, 1, h, s, d, dt=F32) for i, h in enumerate((hq, hkv, hkv, hq)))
    q[0, 1, 70, 3] = NAN
    k[0, 1, 150, 5] = NAN          # seen by rows 150..179 of heads 2 and 3
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    mask = torch.ones(1, 1, s, s, dtype=torch.bool, device=DEV) if masked else None
    out = ax.flash_attention(q, k, v, score_mod=ax.sink_window_mod(30, 4), mask=mask)
    dq, = torch.autograd.grad(out, q, do)
    want = torch.zeros(1, hq, s, dtype=torch.bool, device=DEV)
    want[0, 1, 70] = True
    want[0, 2:, 150:180] = True
    assert torch.equal(out.isnan().any(-1), want) and torch.equal(out.isnan().all(-1), want)
    # dQ = dS K: where dS is 0 a NaN in K still makes the product NaN, so heads 2 and 3 may hold more
    assert bool(dq.isnan().all(-1)[want].all())
    assert torch.equal(dq.isnan().any(-1)[:, :2], want[:, :2])


@pytest.mark.parametrize("t", [6, 20, 70])
def test_padding_parents_are_not_looked_at(t):
    """What stands behind a tree's length is padding: any parents, no notice."""
    lens, tl = [100, 40], [t // 2, t]
    cache = make_cache(2, lens, 1, 128, 16, BF)
    q, dk, dv = randn(1, 2, 4, t, 128), randn(2, 2, 1, t, 128), randn(3, 2, 1, t, 128)
    par = random_tree(5, 2, t)
    wild = par.clone()
    wild[0, tl[0]:] = torch.arange(t - tl[0]).to(torch.int32) + 1000
    assert _lib.device_status() == 0
    got = ax.paged_tree_attention(q, dk, dv, cache, wild, tree_lengths=tl)
    assert _lib.device_status() == 0
    check_tree(cache, lens, q, dk, dv, par, tl, got)


def test_indices_wider_than_32_bits_on_the_device():
    """64-bit indices on the device that 32 bits do not hold are out of range, not their low half."""
    cache = make_cache(1, [40, 20], 1, 64, 16, BF)
    kp, vp, table = cache.key_pool.clone(), cache.value_pool.clone(), cache.block_table.clone()
    far = (1 << 32) + 1
    mk = lambda *x: torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
    assert _lib.device_status() == 0
    ax.copy_blocks(cache, mk(0, far), mk(far, 2))
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    assert torch.equal(cache.key_pool.nan_to_num(7), kp.nan_to_num(7))
    assert torch.equal(cache.value_pool.nan_to_num(7), vp.nan_to_num(7))
    out, freed, count = ax.free_sequences(cache, mk(far))
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    assert torch.equal(out.block_table, table) and int(count) == 0
    # parents and accepted drafts from the host
    t = 4
    q, dk, dv = randn(1, 2, 2, t, 64), randn(2, 2, 1, t, 64), randn(3, 2, 1, t, 64)
    par = torch.tensor([[-1, 1 << 32, -(1 << 32), 2], [-1, 0, 0, 0]])
    good = torch.tensor([[-1, -1, -1, 2], [-1, 0, 0, 0]], dtype=torch.int32)
    got = ax.paged_tree_attention(q, dk, dv, cache, par)
    assert _lib.device_status() == _lib.NOTICE_TREE_ORDER
    check_tree(cache, [40, 20], q, dk, dv, good, [t, t], got)
    with pytest.raises(ValueError):
        ax.append_accepted(cache, dk, dv, [[1 << 32], [0]], [1, 1])


def test_overlong_sequences_are_refused_on_other_caches():
    """A length past its table row raises for the caches that are gathered, as for the others."""
    cache = make_cache(5, [45, 30], 2, 32, 4, F32)
    wrong = ax.PagedKVCache(cache.key_pool, cache.value_pool, cache.block_table,
                            torch.tensor([45 + 4, 30], dtype=torch.int32, device=DEV))
    q = randn(6, 2, 4, 2, 32, dt=F32)
    with pytest.raises(ValueError):
        ax.paged_window_attention(q, wrong, window_size=21, num_sinks=2)
    with pytest.raises(ValueError):
        ax.paged_tree_attention(q, q[:, :2], q[:, :2], wrong, [[-1, 0]] * 2)


def test_fork_with_an_id_listed_twice_on_the_device():
    """The first fork has the page; the second keeps its full pages, as with an id that is no page."""
    lens, bs = [37, 20, 5, 0, 0, 0], 16
    g = torch.Generator().manual_seed(1)
    pools = [torch.randn(20, bs, 1, 64, generator=g).to(BF).to(DEV) for _ in range(2)]
    table = torch.tensor([[0, 1, 2], [3, 4, -1], [5, -1, -1], [-1] * 3, [-1] * 3, [-1] * 3], dtype=torch.int32)
    cache = ax.PagedKVCache(*pools, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    k, v = cache.key_pool.clone(), cache.value_pool.clone()
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    assert _lib.device_status() == 0
    out, used = ax.fork_sequences(cache, mk([0, 1, 2]), mk([3, 4, 5]), mk([9, 9, 10]))
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    assert int(used) == 3
    assert out.block_table[3:].tolist() == [[0, 1, 9], [3, -1, -1], [10, -1, -1]]
    assert out.seq_lengths.tolist() == [37, 20, 5, 37, 16, 5]
    for a, b in ((2, 9), (5, 10)):
        k[b], v[b] = k[a], v[a]
    assert torch.equal(cache.key_pool, k) and torch.equal(cache.value_pool, v)


def _odd_pools(kind, nb, bs, hkv, d, dt):
    """Pools that are not contiguous, or contiguous at an odd address."""
    g = torch.Generator(device=DEV).manual_seed(nb)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)  # noqa: E731
    if kind == "interleaved":          # K and V of a page side by side
        both = mk(nb, 2, bs, hkv, d)
        return both[:, 0], both[:, 1]
    if kind == "head major":
        return tuple(mk(nb, hkv, bs, d).transpose(1, 2) for _ in range(2))
    return tuple(mk(nb * bs * hkv * d + 1)[1:].view(nb, bs, hkv, d) for _ in range(2))


@pytest.mark.parametrize("kind", ["interleaved", "head major", "odd address"])
@pytest.mark.parametrize("d,bs,dt", [(128, 16, BF), (64, 32, HF), (32, 4, F32)])
def test_pools_of_other_layouts(kind, d, bs, dt):
    """Windows, trees, gathers and decodes read such pools where their tokens are."""
    lens, hq, hkv, t = [45, 0, 70], 4, 2, 3
    kp, vp = _odd_pools(kind, 30, bs, hkv, d, dt)
    table = torch.randperm(30, generator=torch.Generator().manual_seed(1)).to(torch.int32)[:3 * (30 // 3)].view(3, -1)
    table = torch.cat([table, table[:, :10].flip(0)], 1)[:, :18]   # (rows may share pages)
    cache = ax.PagedKVCache(kp, vp, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))
    q = randn(1, 3, hq, t, d, dt=dt)
    check_window(cache, lens, q, ax.paged_window_attention(q, cache, window_size=21, num_sinks=2), 21, 2)
    dk, dv, par = randn(2, 3, hkv, t, d, dt=dt), randn(3, 3, hkv, t, d, dt=dt), random_tree(4, 3, t)
    check_tree(cache, lens, q, dk, dv, par, [t] * 3, ax.paged_tree_attention(q, dk, dv, cache, par))
    full = ax.paged_attention_batched(q, cache)
    for i, n in enumerate(lens):
        k, v = history(cache, i, n)
        keys, values, m = ax.gather_kv(cache, i)
        assert m == n and torch.equal(keys, k[0].transpose(0, 1)) and torch.equal(values, v[0].transpose(0, 1))
        if n == 0:
            assert float(full[i].abs().max()) == 0.0
            continue
        want, bound = attention64(q[i:i + 1], k, v, torch.ones(t, n, dtype=torch.bool, device=DEV))
        assert_within(full[i:i + 1], want, bound, "decode")


@pytest.mark.parametrize("kind", ["interleaved", "head major"])
def test_appending_needs_contiguous_pools(kind):
    """What is written in place is not written to where it does not belong."""
    kp, vp = _odd_pools(kind, 6, 16, 2, 64, BF)
    cache = ax.PagedKVCache(kp, vp, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV),
                            torch.tensor([3], dtype=torch.int32, device=DEV))
    before = kp.clone()
    with pytest.raises(ValueError, match="contiguous"):
        ax.append_kv(cache, 0, randn(1, 2, 2, 64), randn(2, 2, 2, 64))
    assert torch.equal(kp, before)


def test_appending_at_an_odd_address():
    kp, vp = _odd_pools("odd address", 6, 16, 2, 64, BF)
    cache = ax.PagedKVCache(kp, vp, torch.tensor([[4, 1]], dtype=torch.int32, device=DEV),
                            torch.tensor([3], dtype=torch.int32, device=DEV))
    k, v = randn(1, 20, 2, 64), randn(2, 20, 2, 64)
    want = kp.clone()
    want[4, 3:], want[1, :7] = k[:13], k[13:]
    out = ax.append_kv(cache, 0, k, v)
    assert torch.equal(out.key_pool, want) and out.seq_lengths.tolist() == [23]
