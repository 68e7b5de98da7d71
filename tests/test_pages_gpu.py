"""The page operators against the same steps on host tables, entry by entry, and a serving loop of all of them."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests._plain64 import assert_within, attention64
from tests.test_paged_rows_gpu import history, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rand_cache(seed, lens, hkv, d, bs, dt, spare=5, width=0, room=0):
    """Random pools and pages; returns the cache and the ids that no row holds."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + room) // bs) for n in lens]
    nb = sum(need) + spare
    perm = torch.randperm(nb, generator=g).tolist()
    table = torch.full((len(lens), max(max(need), 1) + width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
        at += n
    pools = [torch.randn(nb, bs, hkv, d, generator=g).to(dt).to(DEV) for _ in range(2)]
    return ax.PagedKVCache(*pools, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)), perm[at:]


def host(cache):
    return (cache.key_pool.cpu().clone(), cache.value_pool.cpu().clone(), cache.block_table.tolist(),
            cache.seq_lengths.tolist())


def check(cache, k, v, table, lens):
    assert torch.equal(cache.key_pool.cpu(), k) and torch.equal(cache.value_pool.cpu(), v)
    assert cache.block_table.tolist() == table
    assert cache.seq_lengths.tolist() == lens


SHAPES = [(2, 128, 16, BF), (8, 64, 32, HF), (1, 3, 5, BF), (3, 7, 4, F32), (1, 2, 1, HF)]


@pytest.mark.parametrize("hkv,d,bs,dt", SHAPES)
@pytest.mark.parametrize("device", ["cpu", DEV])
def test_copy(hkv, d, bs, dt, device):
    cache, _ = rand_cache(1, [50], hkv, d, bs, dt, spare=60)
    k, v, table, lens = host(cache)
    perm = torch.randperm(cache.num_blocks, generator=torch.Generator().manual_seed(3))
    src, dst = perm[:25].to(torch.int32), perm[25:50].to(torch.int32)
    src[7] = src[3]              # one page to two places
    src[9] = dst[9]              # onto itself
    k[dst.long()], v[dst.long()] = k[src.long()], v[src.long()]
    out = ax.copy_blocks(cache, src.to(device), dst.to(device))
    check(out, k, v, table, lens)
    assert _lib.device_status() == 0


def test_copy_skips_what_it_cannot_do():
    """On the device: out of range, a destination named again, a page that is source and destination."""
    cache, _ = rand_cache(1, [16], 1, 64, 16, BF, spare=30)
    k, v, table, lens = host(cache)
    nb = cache.num_blocks
    src = torch.tensor([0, 1, -1, 4, nb, 6, 7, 2], dtype=torch.int32, device=DEV)
    dst = torch.tensor([10, 10, 11, nb + 3, 12, 7, 13, 14], dtype=torch.int32, device=DEV)
    for s, t in ((0, 10), (7, 13), (2, 14)):
        k[t], v[t] = k[s], v[s]
    ax.copy_blocks(cache, src, dst)
    check(cache, k, v, table, lens)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST


def test_copy_long_lists():
    """Many entries share their look through the lists; the rules stay."""
    cache, _ = rand_cache(1, [1], 1, 8, 1, BF, spare=4000)
    k, v, table, lens = host(cache)
    nb = cache.num_blocks
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    src, dst = perm[:1999].clone(), perm[1999:3998].clone()
    src[500], dst[1300], src[77] = nb, -5, dst[77]    # skipped, skipped, onto itself
    dst[1501] = dst[1500]                             # the first wins
    src[1998] = dst[40]                               # entry 40 may not write a source
    ok = [i for i in range(1999) if i not in (500, 1300, 77, 1501, 40)]
    k[dst[ok].long()], v[dst[ok].long()] = k[src[ok].long()], v[src[ok].long()]
    out = ax.copy_blocks(cache, src.to(DEV), dst.to(DEV))
    check(out, k, v, table, lens)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST


def fork_model(bs, table, lens, src, dst, free):
    """(table, lens, page copies, used) of the forks, one after the other on the old table."""
    new, newlen, moves, used = [list(r) for r in table], list(lens), [], 0
    for s, t in zip(src, dst):
        n = -(-lens[s] // bs)
        new[t] = table[s][:n] + [-1] * (len(table[s]) - n)
        newlen[t] = lens[s]
        if lens[s] % bs:
            moves.append((table[s][n - 1], free[used]))
            new[t][n - 1] = free[used]
            used += 1
    return new, newlen, moves, used


@pytest.mark.parametrize("hkv,d,bs,dt", SHAPES)
@pytest.mark.parametrize("device", ["cpu", DEV])
def test_fork(hkv, d, bs, dt, device):
    lens = [37, 32, 1, 0, 9, 0, 64, 3]
    cache, free = rand_cache(2, lens, hkv, d, bs, dt, spare=9, width=2)
    k, v, table, lens = host(cache)
    src, dst = [0, 1, 0, 2, 3, 5], [3, 5, 7, 4, 6, 1]   # rows that are source and destination, an empty source
    want, wlens, moves, used = fork_model(bs, table, lens, src, dst, free)
    for a, b in moves:
        k[b], v[b] = k[a], v[a]
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    before = cache.block_table.clone()
    out, n = ax.fork_sequences(cache, mk(src), mk(dst), mk(free))
    check(out, k, v, want, wlens)
    assert int(n) == used and n.dtype == torch.int32 and n.is_cuda
    assert torch.equal(cache.block_table, before)      # the old cache's table is as it was
    assert _lib.device_status() == 0


def test_fork_with_exactly_enough_and_too_few_ids():
    cache, free = rand_cache(2, [17, 16, 5, 0, 0], 1, 64, 16, BF, spare=9)
    out, n = ax.fork_sequences(cache, [0, 1], [3, 4], free[:1])   # only the first has an open page
    assert int(n) == 1 and out.seq_lengths.tolist() == [17, 16, 5, 17, 16]
    with pytest.raises(ValueError):
        ax.fork_sequences(cache, [0, 2], [3, 4], free[:1])
    none, n = ax.fork_sequences(cache, [1], [3], [])
    assert int(n) == 0 and none.seq_lengths.tolist() == [17, 16, 5, 16, 0]
    same, n = ax.fork_sequences(cache, [], [], free)
    assert int(n) == 0 and same is cache


def test_fork_skips_what_it_cannot_do():
    cache, free = rand_cache(2, [17, 16, 5, 0, 0, 0], 1, 64, 16, BF, spare=9)
    k, v, table, lens = host(cache)
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    # row 3 twice (the first wins, both take an id), rows out of range, an id that is no page
    out, n = ax.fork_sequences(cache, mk([0, 2, 9, 0, 2]), mk([3, 3, 4, -1, 5]), mk([free[0], free[1], 1000] + free[3:]))
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    p = free[0]
    k[p], v[p] = k[table[0][1]], v[table[0][1]]
    table[3] = [table[0][0], p]
    lens[3] = 17
    table[5], lens[5] = [-1, -1], 0       # its only page could not be copied
    check(out, k, v, table, lens)
    assert int(n) == 3


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("device", ["cpu", DEV])
def test_free(seed, device):
    """Shared pages stay while a row refers to them; the list is ascending."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 200, (9,), generator=g).tolist()
    cache, free = rand_cache(seed, lens, 1, 8, 16, BF, spare=70)
    cache, _ = ax.fork_sequences(cache, [0, 1, 2], [6, 7, 8], free)
    k, v, table, lens = host(cache)
    gone = [0, 7, 4, 8, 2][:seed + 1]
    pages = {p for r in gone for p in table[r] if p >= 0}
    for r in gone:
        table[r], lens[r] = [-1] * len(table[r]), 0
    want = sorted(pages - {p for r in table for p in r})
    out, freed, n = ax.free_sequences(cache, torch.tensor(gone, dtype=torch.int32, device=device))
    check(out, k, v, table, lens)
    assert int(n) == len(want) and freed.tolist() == want + [-1] * (cache.num_blocks - len(want))
    assert _lib.device_status() == 0


def test_free_nothing_twice_and_out_of_range():
    cache, _ = rand_cache(1, [20, 33], 1, 8, 16, BF)
    k, v, table, lens = host(cache)
    out, freed, n = ax.free_sequences(cache, [])
    check(out, k, v, table, lens)
    assert int(n) == 0 and set(freed.tolist()) == {-1}
    out, freed, n = ax.free_sequences(cache, [1, 1])
    assert int(n) == 3 and out.seq_lengths.tolist() == [20, 0]
    out, freed, n = ax.free_sequences(cache, torch.tensor([5, -2], dtype=torch.int32, device=DEV))
    check(out, k, v, table, lens)
    assert int(n) == 0 and _lib.device_status() == _lib.NOTICE_PAGE_LIST


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (40, 17), (500, 0), (33, 1000)])
def test_free_window(window, sinks):
    bs, lens = 16, [200, 0, 16, 17, 31, 65]
    cache, _ = rand_cache(4, lens, 1, 8, bs, BF)
    k, v, table, lens = host(cache)
    gone = []
    for r, n in enumerate(lens):
        for c, p in enumerate(table[r]):
            # the next token stands at n and sees n - window + 1 .. n, and the sinks
            if p >= 0 and all(t >= sinks and n - t >= window for t in range(c * bs, (c + 1) * bs)):
                gone.append(p)
                table[r][c] = -1
    out, freed, n = ax.free_window(cache, window_size=window, num_sinks=sinks)
    check(out, k, v, table, lens)
    assert freed.tolist() == sorted(gone) + [-1] * (cache.num_blocks - len(gone)) and int(n) == len(gone)


@pytest.mark.parametrize("seed", range(5))
@pytest.mark.parametrize("hkv,d,bs,dt", SHAPES)
def test_compact(seed, hkv, d, bs, dt):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, 90, (7,), generator=g).tolist()
    if seed == 4:
        lens = [0] * 7
    cache, free = rand_cache(seed, lens, hkv, d, bs, dt, spare=[0, 40, 1, 300, 5][seed])
    k, v, table, lens = host(cache)
    if seed == 3:                               # a row that shares another's pages, and pages given up in the middle
        table[6] = list(table[0])
        table[1][:2] = [-1, -1]
        cache = ax.PagedKVCache(cache.key_pool, cache.value_pool, torch.tensor(table, dtype=torch.int32, device=DEV),
                                cache.seq_lengths)
    live = sorted({p for r in table for p in r if p >= 0})
    holes = [p for p in range(len(live)) if p not in live]
    to = dict(zip([p for p in live if p >= len(live)], holes))
    for a, b in to.items():
        k[b], v[b] = k[a], v[a]
    out, n = ax.compact_blocks(cache)
    check(out, k, v, [[to.get(p, p) for p in r] for r in table], lens)
    assert int(n) == len(live)
    again, n2 = ax.compact_blocks(out)           # nothing left to move
    check(again, k, v, out.block_table.tolist(), lens)
    assert int(n2) == len(live)


@pytest.mark.parametrize("hkv,d,bs,dt", SHAPES)
@pytest.mark.parametrize("chk", [True, False])
def test_append_accepted(hkv, d, bs, dt, chk):
    lens, t, a = [0, 15, 16, 33, 7], 9, 6
    cache, _ = rand_cache(6, lens, hkv, d, bs, dt, room=a)
    k, v, table, lens = host(cache)
    dk, dv = (randn(s, 5, t, hkv, d, dt=dt).transpose(1, 2) for s in (1, 2))
    acc = torch.stack([torch.randperm(t, generator=torch.Generator().manual_seed(i))[:a] for i in range(5)])
    acc[2, 1] = acc[2, 0]                        # one draft twice
    n = [6, 0, 3, 1, 6]
    for s in range(5):
        for i in range(n[s]):
            pos = lens[s] + i
            k[table[s][pos // bs], pos % bs] = dk[s, :, acc[s, i]].cpu()
            v[table[s][pos // bs], pos % bs] = dv[s, :, acc[s, i]].cpu()
    for s in range(5):                           # what lies behind the count is not read
        acc[s, n[s]:] = 10000
    out = ax.append_accepted(cache, dk, dv, acc, n, check=chk)
    check(out, k, v, table, [x + y for x, y in zip(lens, n)])
    assert cache.seq_lengths.tolist() == lens and _lib.device_status() == 0


def test_append_accepted_refuses_or_skips():
    lens = [14, 20, 3]
    cache, _ = rand_cache(6, lens, 1, 64, 16, BF, room=3)     # row 0 has a page for 14 + 2 + .. tokens, row 2 one page
    k, v, table, lens = host(cache)
    dk, dv = randn(1, 3, 1, 4, 64), randn(2, 3, 1, 4, 64)
    acc = torch.tensor([[0, 1, 2, 3], [3, 9, 1, 0], [2, 1, 0, 0]], dtype=torch.int32)
    for n in ([4, 2, 0], [0, 2, 0], [0, 0, -1], [0, 0, 5]):
        with pytest.raises(ValueError):
            ax.append_accepted(cache, dk, dv, acc, n)
        check(cache, k, v, table, lens)
    assert _lib.device_status() == 0
    out = ax.append_accepted(cache, dk, dv, acc, [1, 2, 9], check=False)
    assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
    rows = [(0, 14, 0), (1, 20, 3)] + [(2, 3 + i, int(acc[2, i])) for i in range(4)]
    for s, pos, tok in rows:
        k[table[s][pos // 16], pos % 16] = dk[s, :, tok].cpu()
        v[table[s][pos // 16], pos % 16] = dv[s, :, tok].cpu()
    check(out, k, v, table, [15, 22, 7])


@pytest.mark.parametrize("nb,rows", [(819200, 3), (819201, 3), (1200000, 400)])
def test_sets_of_many_pages(nb, rows):
    """Pools on both sides of what the bit maps in shared memory hold."""
    g = torch.Generator().manual_seed(nb)
    pool = torch.arange(nb, dtype=torch.float32, device=DEV).view(nb, 1, 1, 1)
    ids = torch.randperm(nb, generator=g)[:rows * 700].view(rows, 700).to(torch.int32)
    ids[0, 0], ids[1, 3] = nb - 1, 0
    cache = ax.PagedKVCache(pool, pool.clone(), ids.to(DEV), torch.full((rows,), 700, dtype=torch.int32, device=DEV))
    out, freed, n = ax.free_sequences(cache, [0, rows - 1])
    left = set(ids[1:rows - 1].flatten().tolist())
    want = sorted(set(ids[[0, rows - 1]].flatten().tolist()) - left)
    assert int(n) == len(want) and freed[:len(want)].tolist() == want and bool((freed[len(want):] == -1).all())
    new, live = ax.compact_blocks(out)
    assert int(live) == len(left)
    t, old = new.block_table[1:rows - 1].cpu(), ids[1:rows - 1]
    assert sorted(set(t.flatten().tolist())) == list(range(len(left)))
    assert torch.equal(new.key_pool.flatten()[t.to(DEV).long()].cpu().to(torch.int32), old)
    assert torch.equal(new.value_pool.flatten()[t.to(DEV).long()].cpu().to(torch.int32), old)
    stay = old < len(left)
    assert torch.equal(t[stay], old[stay])


def test_pools_past_32_bits():
    """More than 2^31 elements: the last pages are copied, forked, compacted and appended where they are."""
    bs, hkv, d = 256, 16, 128
    nb = (1 << 31) // (bs * hkv * d) + 6
    kp = torch.zeros(nb, bs, hkv, d, dtype=BF, device=DEV)
    vp = torch.zeros_like(kp)
    kp[-3:], vp[-3:] = randn(1, 3, bs, hkv, d), randn(2, 3, bs, hkv, d)
    k3, v3 = kp[-3:].clone(), vp[-3:].clone()
    cache = ax.PagedKVCache(kp, vp, torch.tensor([[nb - 1, nb - 2], [-1, -1]], dtype=torch.int32, device=DEV),
                            torch.tensor([300, 0], dtype=torch.int32, device=DEV))
    ax.copy_blocks(cache, [nb - 3], [nb - 5])
    assert torch.equal(kp[-5], k3[0]) and torch.equal(vp[-5], v3[0])
    out, _ = ax.fork_sequences(cache, [0], [1], [nb - 4])
    assert torch.equal(kp[-4], k3[1]) and torch.equal(vp[-4], v3[1])
    dk, dv = randn(3, 2, hkv, 2, d), randn(4, 2, hkv, 2, d)
    out = ax.append_accepted(out, dk, dv, [[1], [0]], [1, 1])
    assert torch.equal(kp[nb - 2, 300 - 256], dk[0, :, 1]) and torch.equal(vp[nb - 4, 300 - 256], dv[1, :, 0])
    out, n = ax.compact_blocks(out)
    assert int(n) == 3 and sorted(out.block_table.flatten().tolist()) == [0, 1, 2, 2]
    assert torch.equal(kp[out.block_table[0, 0]], k3[2]) and torch.equal(vp[out.block_table[0, 0]], v3[2])


def test_captured_and_replayed():
    """Two graphs of the same steps with their own scratch; a replay follows the tables it finds."""
    lens = [40, 33, 17, 0, 0]
    cache, free = rand_cache(9, lens, 2, 64, 16, BF, spare=8)
    src, dst = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 2], [3, 4]))
    ids = torch.tensor(free, dtype=torch.int32, device=DEV)
    ends = torch.tensor([0, 1], dtype=torch.int32, device=DEV)

    def steps():
        a, used = ax.fork_sequences(cache, src, dst, ids)
        b, freed, n = ax.free_sequences(a, ends)
        return a, used, b, freed, n

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        steps()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = steps()
        graphs.append((g, res))
    ends.copy_(torch.tensor([2, 4], dtype=torch.int32))
    src.copy_(torch.tensor([1, 2], dtype=torch.int32))
    for g, _ in graphs:
        g.replay()
    table, lens = cache.block_table.tolist(), cache.seq_lengths.tolist()
    want, wlens, moves, used = fork_model(16, table, lens, [1, 2], [3, 4], free)
    for _, (a, n_used, b, freed, n) in graphs:
        assert a.block_table.tolist() == want and a.seq_lengths.tolist() == wlens and int(n_used) == used
        left = {p for r in (0, 1, 3) for p in want[r]}
        gone = sorted({p for r in (2, 4) for p in want[r] if p >= 0} - left)
        assert freed.tolist()[:int(n)] == gone
        assert b.seq_lengths.tolist() == [wlens[0], wlens[1], 0, wlens[3], 0]


def test_serving_loop():
    """Prompts, forks, drafted trees, accepted paths, window decode, freeing and compaction: after every
    step the attention over the pages equals the formula on each sequence's own history."""
    hkv, hq, d, bs, window, sinks, nb, t = 2, 8, 128, 16, 48, 4, 96, 6
    cache = ax.init_paged_kv_cache(num_blocks=nb, block_size=bs, num_kv_heads=hkv, head_dim=d, batch_size=4,
                                   max_blocks_per_seq=16)
    free = list(range(nb))
    hist = [[torch.zeros(0, hkv, d, device=DEV, dtype=BF)] * 2 for _ in range(4)]
    for i, n in ((0, 70), (1, 33)):
        cache, used = ax.allocate_blocks(cache, sequence_idx=i, num_new_tokens=n, free_block_ids=free)
        free = free[used:]
        kv = [randn(10 * i + s, n, hkv, d) for s in (0, 1)]
        cache = ax.append_kv(cache, i, *kv)
        hist[i] = kv
    cache, used = ax.fork_sequences(cache, [0, 0], [2, 3], free)
    free = free[int(used):]
    hist[2], hist[3] = list(hist[0]), list(hist[0])
    for step in range(5):
        q = randn(100 + step, 4, hq, t, d)
        dk, dv = randn(200 + step, 4, hkv, t, d), randn(300 + step, 4, hkv, t, d)
        par = torch.tensor([[-1, 0, 1, 0, 3, -1]] * 4, dtype=torch.int32)
        got = ax.paged_tree_attention(q, dk, dv, cache, par, max_context=256)
        for i in range(4):
            see = torch.zeros(t, len(hist[i][0]) + t, dtype=torch.bool)
            see[:, :len(hist[i][0])] = True
            for r in range(t):
                p = r
                while p >= 0:
                    see[r, len(hist[i][0]) + p] = True
                    p = int(par[i, p])
            k, v = (torch.cat([h, x[i].transpose(0, 1)]).permute(1, 0, 2)[None] for h, x in zip(hist[i], (dk, dv)))
            want, bound = attention64(q[i:i + 1], k, v, see.to(DEV))
            assert_within(got[i:i + 1], want, bound, f"step {step} tree {i}")
        path, n = [[0, 1, 2], [5, 0, 0], [0, 3, 4], [0, 3, 0]], [3, 1, 3, 2]
        for i in range(4):
            cache, used = ax.allocate_blocks(cache, sequence_idx=i, num_new_tokens=n[i], free_block_ids=free)
            free = free[used:]
            hist[i] = [torch.cat([h, x[i].transpose(0, 1)[path[i][:n[i]]]]) for h, x in zip(hist[i], (dk, dv))]
        cache = ax.append_accepted(cache, dk, dv, path, n)
        q1 = randn(400 + step, 4, hq, 1, d)
        got = ax.paged_window_attention(q1, cache, window_size=window, num_sinks=sinks, max_context=256)
        for i in range(4):
            m = len(hist[i][0])
            col = torch.arange(m, device=DEV)[None]
            keep = (m - 1 - col < window) | (col < sinks)
            k, v = (h.permute(1, 0, 2)[None] for h in hist[i])
            want, bound = attention64(q1[i:i + 1], k, v, keep)
            assert_within(got[i:i + 1], want, bound, f"step {step} window {i}")
    # the window's users give up far pages; then a row ends and the pool is packed
    slim, freed, n = ax.free_window(cache, window_size=window, num_sinks=sinks)
    assert int(n) > 0
    a = ax.paged_window_attention(q1, slim, window_size=window, num_sinks=sinks, max_context=256)
    assert torch.equal(a, got)
    cache, freed, n = ax.free_sequences(cache, [0])
    free = free + freed.tolist()[:int(n)]
    cache, live = ax.compact_blocks(cache)
    assert int(live) + len(free) == nb
    for i in (1, 2, 3):
        k, v = history(cache, i, len(hist[i][0]))
        assert torch.equal(k[0].permute(1, 0, 2), hist[i][0]) and torch.equal(v[0].permute(1, 0, 2), hist[i][1])
    assert _lib.device_status() == 0
