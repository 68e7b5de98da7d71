"""paged_window_attention and paged_tree_attention against the formula in 64 bits."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make_cache(seed, lens, hkv, d, bs, dt, width=None):
    """Random pages at random places; slots that hold no token are NaN, and so is the pool's last page."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + 3
    perm = torch.randperm(nb - 1, generator=g).to(torch.int32)
    width = width or max(max(need), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    kp = torch.randn(nb, bs, hkv, d, generator=g).to(dt)
    vp = torch.randn(nb, bs, hkv, d, generator=g).to(dt)
    at = 0
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
        for c in range(n):
            used[table[i, c], :max(0, min(bs, lens[i] - c * bs))] = True
    kp[~used], vp[~used] = float("nan"), float("nan")
    return ax.PagedKVCache(kp.to(DEV), vp.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV))


def history(cache, i, n):
    bs = cache.block_size
    pages = cache.block_table[i, :-(-n // bs)].long()
    cut = lambda pool: pool[pages].flatten(0, 1)[:n].permute(1, 0, 2)[None]  # noqa: E731
    return cut(cache.key_pool), cut(cache.value_pool)


def randn(seed, *shape, dt=BF):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dt)


def check_window(cache, lens, q, got, window, sinks):
    t = q.shape[2]
    for i, n in enumerate(lens):
        if n == 0:
            assert float(got[i].abs().max()) == 0.0
            continue
        k, v = history(cache, i, n)
        row = torch.arange(n - t, n, device=DEV)[:, None]
        col = torch.arange(n, device=DEV)[None]
        keep = (col <= row) & ((row - col < window) | (col < sinks))
        want, bound = attention64(q[i:i + 1], k, v, keep)
        assert_within(got[i:i + 1], want, bound, f"sequence {i} (length {n})")


WINDOW = [
    # lens, hq, hkv, d, page, dtype, T, window, sinks
    ([1, 2, 17, 300, 0], 8, 2, 128, 16, BF, 1, 64, 4),
    ([700, 4096, 33], 4, 4, 128, 16, HF, 1, 200, 0),
    ([1000, 15, 5000], 8, 1, 64, 32, BF, 1, 1000, 17),
    ([900, 3, 40], 6, 2, 128, 48, BF, 5, 1, 1),        # a window of one, rows in front of the short sequence
    ([2049, 2048, 2047, 129], 4, 2, 128, 64, HF, 7, 333, 130),
    ([600, 610], 8, 2, 64, 16, HF, 9, 100, 5),         # 36 rows: four row tiles
    ([500, 77], 16, 2, 128, 128, BF, 16, 250, 40),     # 128 rows
    ([3000], 12, 4, 128, 256, BF, 3, 100000, 4),       # window beyond the sequence: causal decode
    ([20000], 4, 1, 128, 16, BF, 1, 64, 1),            # far sinks: two pages of many
    ([5000, 1], 2, 2, 64, 96, BF, 2, 17, 9000),        # more sinks than tokens
    ([321, 9], 32, 1, 128, 16, HF, 40, 70, 3),         # 1280 rows of one kv head
]


@pytest.mark.parametrize("lens,hq,hkv,d,bs,dt,t,window,sinks", WINDOW)
def test_window(lens, hq, hkv, d, bs, dt, t, window, sinks):
    cache = make_cache(len(lens) + t, lens, hkv, d, bs, dt)
    q = randn(t, len(lens), hq, t, d, dt=dt)
    got = ax.paged_window_attention(q, cache, window_size=window, num_sinks=sinks)
    check_window(cache, lens, q, got, window, sinks)
    # the same without a host sync, from a loose bound
    again = ax.paged_window_attention(q, cache, window_size=window, num_sinks=sinks,
                                      max_context=cache.block_table.shape[1] * bs)
    check_window(cache, lens, q, again, window, sinks)
    assert _lib.device_status() == 0


def test_window_needs_only_its_pages():
    """Pages outside the window and the sinks may be gone: their entries are -1 and the page they
    would select holds NaN."""
    lens, window, sinks, bs = [1000, 317, 64], 100, 20, 16
    cache = make_cache(3, lens, 2, 128, bs, BF)
    table = cache.block_table.clone()
    for i, n in enumerate(lens):
        for c in range(-(-n // bs)):
            if c * bs >= sinks and (c + 1) * bs <= n - window:
                table[i, c] = -1
    assert int((table == -1).sum()) > int((cache.block_table == -1).sum())
    q = randn(1, 3, 8, 1, 128)
    got = ax.paged_window_attention(q, ax.PagedKVCache(cache.key_pool, cache.value_pool, table, cache.seq_lengths),
                                    window_size=window, num_sinks=sinks)
    check_window(cache, lens, q, got, window, sinks)


@pytest.mark.parametrize("d,bs,dt", [(32, 4, F32), (128, 12, BF), (128, 16, F32)])
def test_window_other_caches(d, bs, dt):
    """Caches that the fused kernel does not take go through the flash kernel."""
    lens = [45, 3, 0, 130]
    cache = make_cache(5, lens, 2, d, bs, dt)
    q = randn(6, 4, 4, 4, d, dt=dt)
    check_window(cache, lens, q, ax.paged_window_attention(q, cache, window_size=21, num_sinks=2), 21, 2)


def random_tree(seed, b, t, chain=False):
    g = torch.Generator().manual_seed(seed)
    par = torch.full((b, t), -1, dtype=torch.int32)
    for i in range(1, t):
        par[:, i] = i - 1 if chain else torch.randint(-1, i, (b,), generator=g).to(torch.int32)
    return par


def check_tree(cache, lens, q, dk, dv, par, tl, got):
    t = q.shape[2]
    for i, n in enumerate(lens):
        m = tl[i]
        if m < t:
            assert float(got[i, :, m:].abs().max()) == 0.0, f"padding rows of sequence {i}"
        if m == 0:
            continue
        see = torch.zeros(m, n + m, dtype=torch.bool)
        see[:, :n] = True
        for r in range(m):
            p = r
            while p >= 0:
                see[r, n + p] = True
                p = int(par[i, p])
        k, v = history(cache, i, n)
        k, v = torch.cat([k, dk[i:i + 1, :, :m]], 2), torch.cat([v, dv[i:i + 1, :, :m]], 2)
        want, bound = attention64(q[i:i + 1, :, :m], k, v, see.to(DEV))
        assert_within(got[i:i + 1, :, :m], want, bound, f"sequence {i} (context {n}, tree {m})")


TREE = [
    # lens, hq, hkv, d, page, dtype, T, chain
    ([100, 0, 17, 1], 8, 2, 128, 16, BF, 1, False),     # one draft; an empty context
    ([257, 700, 16], 4, 1, 128, 16, HF, 4, False),
    ([1000, 31], 8, 2, 64, 32, BF, 7, True),
    ([2048, 2049, 5], 4, 2, 128, 64, BF, 13, False),    # 26 rows
    ([640, 77], 8, 2, 128, 16, HF, 16, False),          # 64 rows
    ([1500], 2, 2, 64, 48, HF, 64, True),               # 64 tokens in one chain
    ([900, 128, 127], 8, 1, 128, 16, BF, 33, False),    # 264 rows of one kv head
    ([500, 0], 16, 2, 64, 128, BF, 65, False),
    ([300, 5], 4, 2, 128, 16, HF, 130, False),          # more drafted tokens than a tile
    ([200], 2, 1, 128, 32, BF, 300, True),
    ([5000], 12, 4, 128, 256, BF, 21, False),
]


@pytest.mark.parametrize("lens,hq,hkv,d,bs,dt,t,chain", TREE)
@pytest.mark.parametrize("padded", [False, True])
def test_tree(lens, hq, hkv, d, bs, dt, t, chain, padded):
    b = len(lens)
    cache = make_cache(t, lens, hkv, d, bs, dt)
    q = randn(1, b, hq, t, d, dt=dt)
    # the projections' layout: (batch, token, head, dim)
    dk, dv = (randn(s, b, t, hkv, d, dt=dt).transpose(1, 2) for s in (2, 3))
    par = random_tree(t, b, t, chain)
    tl = [t] * b
    if padded:
        tl = [t - i * (t + 1) // 2 if t - i * (t + 1) // 2 > 0 else 0 for i in range(1, b + 1)]
        for i, m in enumerate(tl):  # whatever stands in the padding
            q[i, :, m:], dk[i, :, m:], dv[i, :, m:] = float("nan"), float("nan"), float("nan")
            par[i, m:] = -1
    got = ax.paged_tree_attention(q, dk, dv, cache, par.to(DEV), tree_lengths=tl if padded else None)
    check_tree(cache, lens, q, dk, dv, par, tl, got)
    loose = ax.paged_tree_attention(q, dk, dv, cache, par.to(DEV), tree_lengths=tl if padded else None,
                                    max_context=cache.block_table.shape[1] * bs)
    check_tree(cache, lens, q, dk, dv, par, tl, loose)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("d,bs,dt", [(32, 4, F32), (128, 12, BF)])
def test_tree_other_caches(d, bs, dt):
    lens, t = [45, 0, 130], 9
    cache = make_cache(5, lens, 2, d, bs, dt)
    q, dk, dv = (randn(s, 3, h, t, d, dt=dt) for s, h in ((6, 4), (7, 2), (8, 2)))
    par = random_tree(1, 3, t)
    got = ax.paged_tree_attention(q, dk, dv, cache, par, tree_lengths=[9, 4, 0])
    check_tree(cache, lens, q, dk, dv, par, [9, 4, 0], got)


@pytest.mark.parametrize("layout", ["expanded", "odd", "sliced"])
def test_draft_layouts(layout):
    """Drafts broadcast over heads, at an odd address, and as a slice of a wider tensor."""
    lens, t, hkv, d = [70, 5], 5, 2, 128
    cache = make_cache(4, lens, hkv, d, 16, BF)
    q = randn(1, 2, 4, t, d)
    if layout == "expanded":
        dk, dv = (randn(s, 2, 1, t, d).expand(2, hkv, t, d) for s in (2, 3))
    elif layout == "odd":
        dk, dv = (randn(s, 2 * hkv * t * d + 1)[1:].view(2, hkv, t, d) for s in (2, 3))
    else:
        dk, dv = (randn(s, 2, hkv, t, 3 * d)[..., d:2 * d] for s in (2, 3))
    par = random_tree(3, 2, t)
    check_tree(cache, lens, q, dk, dv, par, [t, t], ax.paged_tree_attention(q, dk, dv, cache, par))


def test_parents_out_of_order_are_roots():
    """A parent at or behind its token cannot be on a path: taken as a root, with a notice."""
    lens, t = [50], 6
    cache = make_cache(2, lens, 1, 128, 16, BF)
    q, dk, dv = randn(1, 1, 4, t, 128), randn(2, 1, 1, t, 128), randn(3, 1, 1, t, 128)
    bad = torch.tensor([[0, 5, 1, 2, 100, -7]], dtype=torch.int32)
    good = torch.tensor([[-1, -1, 1, 2, -1, -1]], dtype=torch.int32)
    assert _lib.device_status() == 0
    got = ax.paged_tree_attention(q, dk, dv, cache, bad)
    assert _lib.device_status() == _lib.NOTICE_TREE_ORDER
    check_tree(cache, lens, q, dk, dv, good, [t], got)


def test_lengths_above_the_bound_are_cut_and_noted():
    cache = make_cache(2, [600, 40], 1, 128, 16, BF)
    q = randn(1, 2, 4, 1, 128)
    assert _lib.device_status() == 0
    got = ax.paged_window_attention(q, cache, window_size=5000, max_context=40)
    assert _lib.device_status() == _lib.NOTICE_CONTEXT_OVERRUN
    assert bool(torch.isfinite(got).all())
    # the sequence within the bound is not touched by the other
    k, v = history(cache, 1, 40)
    want, bound = attention64(q[1:2], k, v, torch.ones(1, 40, dtype=torch.bool, device=DEV))
    assert_within(got[1:2], want, bound, "sequence within the bound")


@pytest.mark.parametrize("t", [1, 20])
def test_lengths_past_the_table_row_are_cut_and_noted(t):
    """No more tokens than the row's pages hold: the sequence is read as if it ended there."""
    cache = make_cache(2, [64, 40], 1, 128, 16, BF)
    q = randn(1, 2, 4, t, 128)
    wrong = ax.PagedKVCache(cache.key_pool, cache.value_pool, cache.block_table,
                            torch.tensor([100, 40], dtype=torch.int32, device=DEV))
    assert _lib.device_status() == 0
    got = ax.paged_window_attention(q, wrong, window_size=30, num_sinks=2, max_context=100)
    assert _lib.device_status() == _lib.NOTICE_TABLE_OVERRUN
    check_window(cache, [64, 40], q, got, 30, 2)
    with pytest.raises(ValueError):
        ax.paged_window_attention(q, wrong, window_size=30)


def test_another_stream_and_a_captured_graph():
    """On a side stream, and captured twice into graphs whose replays follow new lengths and queries."""
    lens, window, sinks, t = [300, 129], 64, 4, 3
    cache = make_cache(8, [512, 512], 2, 128, 16, BF)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    cache = ax.PagedKVCache(cache.key_pool, cache.value_pool, cache.block_table, sl)
    q = randn(1, 2, 8, t, 128)
    dk, dv, par = randn(2, 2, 2, t, 128), randn(3, 2, 2, t, 128), random_tree(4, 2, t)
    pd = par.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ax.paged_window_attention(q, cache, window_size=window, num_sinks=sinks, max_context=512)
    torch.cuda.current_stream().wait_stream(side)
    check_window(cache, lens, q, got, window, sinks)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a = ax.paged_window_attention(q, cache, window_size=window, num_sinks=sinks, max_context=512)
            b = ax.paged_tree_attention(q, dk, dv, cache, pd, max_context=512)
        graphs.append((g, a, b))
    for new in ([500, 2], [1, 400]):
        sl.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(randn(new[0], 2, 8, t, 128))
        for g, a, b in graphs:
            g.replay()
        for g, a, b in graphs:
            check_window(cache, new, q, a, window, sinks)
            check_tree(cache, new, q, dk, dv, par, [t, t], b)


def test_wider_query_types_are_cast():
    cache = make_cache(2, [70], 2, 128, 16, BF)
    q = randn(1, 1, 4, 2, 128, dt=F32)
    got = ax.paged_window_attention(q, cache, window_size=30, num_sinks=2)
    assert got.dtype == F32
    check_window(cache, [70], q.to(BF), got.to(BF), 30, 2)


def test_kv_offsets_past_32_bits():
    """A pool of more than 2^31 elements: the last pages are read where they are."""
    bs, hkv, d = 256, 16, 128
    nb = (1 << 31) // (bs * hkv * d) + 5
    kp = torch.zeros(nb, bs, hkv, d, dtype=BF, device=DEV)
    vp = torch.zeros(nb, bs, hkv, d, dtype=BF, device=DEV)
    kp[-2:], vp[-2:] = randn(1, 2, bs, hkv, d), randn(2, 2, bs, hkv, d)
    cache = ax.PagedKVCache(kp, vp, torch.tensor([[nb - 1, nb - 2]], dtype=torch.int32, device=DEV),
                            torch.tensor([300], dtype=torch.int32, device=DEV))
    q = randn(3, 1, 16, 1, d)
    check_window(cache, [300], q, ax.paged_window_attention(q, cache, window_size=200, num_sinks=3), 200, 3)
    dk, dv = randn(4, 1, hkv, 1, d), randn(5, 1, hkv, 1, d)
    par = torch.full((1, 1), -1, dtype=torch.int32)
    check_tree(cache, [300], q, dk, dv, par, [1], ax.paged_tree_attention(q, dk, dv, cache, par))


@pytest.mark.parametrize("d,max_len,dt", [(128, 512, BF), (64, 400, HF), (128, 333, BF), (32, 64, F32)])
@pytest.mark.parametrize("t", [1, 5])
def test_contiguous_cache(d, max_len, dt, t):
    """kv_cache_attention with a window: fused on the buffer, or the flash kernel where that cannot be."""
    b, hq, hkv, n = 2, 4, 2, max_len - 7
    cache = ax.init_kv_layer_cache(b, hkv, d, max_len, dt)
    cache = ax.update_kv_layer_cache(cache, randn(1, b, hkv, n, d, dt=dt), randn(2, b, hkv, n, d, dt=dt), 0)
    q = randn(3, b, hq, t, d, dt=dt)
    got = ax.kv_cache_attention(q, cache, window_size=21, num_sinks=3)
    row, col = torch.arange(n - t, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    keep = (col <= row) & ((row - col < 21) | (col < 3))
    want, bound = attention64(q, cache.keys[:, :, :n], cache.values[:, :, :n], keep)
    assert_within(got, want, bound, "window over a contiguous cache")
    few = ax.KVLayerCache(cache.keys, cache.values, 3)     # more rows than positions
    got = ax.kv_cache_attention(randn(4, b, hq, 5, d, dt=dt), few, window_size=2, num_sinks=0)
    assert float(got[:, :, :2].abs().max()) == 0.0 and bool((got[:, :, 2:] != 0).any())
    mask = (torch.arange(n, device=DEV) % 3 != 0)[None, None, None]
    got = ax.kv_cache_attention(q, cache, window_size=21, num_sinks=3, mask=mask)
    want, bound = attention64(q, cache.keys[:, :, :n], cache.values[:, :, :n], keep & mask[0, 0])
    assert_within(got, want, bound, "and a mask")
