"""Appending batches of tokens to 16-, 32- and 8-bit pages, and gathering them, against 64 bits."""

import dataclasses
import math

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests.test_rotary_gpu import check, turned64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8
BITS8 = (E4M3, INT8)


def make_cache(dt, lens, room, hk=2, d=64, bs=16, seed=0, spare=2):
    """A cache of random values (8-bit pools: random codes, no NaN) whose table covers lens + room."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    need = [-(-(n + room) // bs) for n in lens]
    nb, most = sum(need) + spare, max(max(need), 1)
    perm = torch.randperm(nb, generator=g, device=DEV).int()
    table = torch.full((len(lens), most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    shape = (nb, bs, hk, d)
    if dt not in BITS8:
        k, v = (torch.randn(shape, generator=g, device=DEV).to(dt) for _ in range(2))
        return ax.PagedKVCache(k, v, table, sl)
    k, v = ((torch.randn(shape, generator=g, device=DEV) * 40).clamp(-120, 120).round().to(dt) for _ in range(2))
    ks, vs = (2.0 ** torch.randint(-9, -5, (nb, hk), generator=g, device=DEV).float() for _ in range(2))
    return ax.QuantizedPagedKVCache(k, v, ks, vs, table, sl)


def snapshot(cache):
    return {f.name: getattr(cache, f.name).clone() for f in dataclasses.fields(cache)}


def as_bytes(x):
    return x.view(torch.uint8) if x.dtype == E4M3 else x


def half_of(y, dt, s):
    """Half a step of the 8-bit type around the values y at scale s."""
    if dt == INT8:
        return 0.5 * s + 0 * y
    return torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s + 0 * y)


def check_pools(cache, before, rows, lens, new, dt):
    """Every slot of the pools: new tokens near their 64-bit values, open pages restated, the rest untouched.

    ``rows[name] = (values, bound)`` (B, Hkv, T, D) of the new tokens in 64 bits before the pool's rounding.
    """
    bs = cache.block_size
    most = {E4M3: 448.0, INT8: 127.0}.get(dt)
    for name in ("key", "value"):
        pool, old_pool = getattr(cache, f"{name}_pool"), before[f"{name}_pool"]
        seen = torch.zeros(pool.shape[0], bs, dtype=torch.bool, device=DEV)
        y_all, b_all = rows[name]
        for i, (n, t) in enumerate(zip(lens, new)):
            for p0 in range(n // bs * bs, n + t, bs):
                page = int(cache.block_table[i, p0 // bs])
                lo, hi = max(n, p0), min(n + t, p0 + bs)
                if lo >= hi:
                    continue
                y = y_all[i, :, lo - n:hi - n].transpose(0, 1)
                b = b_all[i, :, lo - n:hi - n].transpose(0, 1)
                seen[page, lo - p0:hi - p0] = True
                if dt not in BITS8:
                    off = (pool[page, lo - p0:hi - p0].double() - y).abs()
                    assert bool((off <= b).all()), f"{name}: {float((off - b).max()):.3e} too far"
                    continue
                seen[page, :lo - p0] = True
                had = lo > p0
                s = getattr(cache, f"{name}_scales")[page].double()
                s_old = before[f"{name}_scales"][page].double() if had else torch.zeros_like(s)
                amax, slack = y.abs().amax((0, 2)), b.amax((0, 2))
                assert bool((torch.frexp(s)[0] == 0.5).all())  # a power of two
                assert bool((s >= s_old).all()) and bool((amax - slack <= most * s).all())
                grown = s > s_old  # then it is the least that will do (2^-100 at least)
                assert bool(((most * s / 2 < amax + slack) | (s == 2.0 ** -100))[grown].all())
                sc = s[:, None]
                off = (pool[page, lo - p0:hi - p0].double() * sc - y).abs()
                lim = half_of(y.abs() + b, dt, sc) + b
                assert bool((off <= lim).all()), f"{name}: {float((off - lim).max()):.3e} too far"
                if had:
                    ratio = (s_old / s).float()[:, None]
                    want = old_pool[page, :lo - p0].float() * ratio
                    want = want.to(E4M3) if dt == E4M3 else want.round().to(INT8)
                    assert torch.equal(as_bytes(pool[page, :lo - p0]), as_bytes(want)), f"{name}: restated codes"
        same = ~seen
        assert torch.equal(as_bytes(pool)[same], as_bytes(old_pool)[same]), f"{name}: an untouched slot changed"


def case(dt, pool, lens, t, new=None, *, hk=2, hq=4, d=64, bs=16, r=None, interleaved=False, seed=0, scale=1.0, **kw):
    torch.manual_seed(seed)
    new = [t] * len(lens) if new is None else new
    cache = make_cache(pool, lens, t, hk, d, bs, seed)
    n = len(lens)
    k, v = ((torch.randn(n, t, hk, d, device=DEV) * scale).to(dt).transpose(1, 2) for _ in range(2))
    q = torch.randn(n, t, hq, d, device=DEV).to(dt).transpose(1, 2)
    r = d if r is None else r
    plan, (w, _) = ax.rotary_plan(r, interleaved=interleaved), ax.rotary_frequencies(r)
    before = snapshot(cache)
    nl = torch.tensor(new, dtype=torch.int32, device=DEV)
    out, q2 = ax.append_tokens(cache, k, v, new_lengths=nl, rotary=plan, query=q, **kw)
    pos = torch.tensor(lens, device=DEV)[:, None] + torch.arange(t, device=DEV)
    check(q2, turned64(q, pos, w, interleaved), "query")
    assert out.seq_lengths.tolist() == [a + b for a, b in zip(lens, new)]
    assert torch.equal(cache.seq_lengths, before["seq_lengths"]) and torch.equal(out.block_table, before["block_table"])
    to = F32 if pool in BITS8 else pool  # (8-bit pools: the bound in front of their own rounding)
    yk, bk = turned64(k.to(F32), pos, w, interleaved)
    if to != F32:
        from tests._plain64 import HALF_STEP, TINY_STEP
        bk = bk + HALF_STEP[to] * (yk.abs() + bk) + TINY_STEP[to]
        bv = HALF_STEP[to] * v.double().abs() + TINY_STEP[to] if to != dt else 0 * v.double()
    else:
        bv = 0 * v.double()
    check_pools(out, before, {"key": (yk, bk), "value": (v.double(), bv)}, lens, new, pool)
    return out


@pytest.mark.parametrize("pool", [BF16, F16, F32, E4M3, INT8])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_types(dt, pool):
    case(dt, pool, [0, 5, 16, 47], 19, [19, 0, 7, 1])


@pytest.mark.parametrize("pool", [BF16, E4M3, INT8])
@pytest.mark.parametrize("kw", [
    dict(lens=[33], t=1, d=128, bs=16), dict(lens=[0, 15, 16, 17], t=1, d=128, hk=8, hq=32),
    dict(lens=[3, 100], t=70, d=128, bs=64, hk=1, hq=3), dict(lens=[7], t=300, d=64, bs=128, hk=3, hq=3),
    dict(lens=[1, 2], t=9, d=80, bs=24, r=40), dict(lens=[5], t=6, d=20, bs=5, r=6, hk=3, hq=3),
    dict(lens=[4, 0], t=33, d=7, bs=8, r=4, hk=1, hq=2), dict(lens=[2000], t=2, d=256, bs=256, hk=2),
    dict(lens=[9, 30], t=40, new=[40, 3], d=96, bs=16, r=48), dict(lens=[0, 0, 0], t=16, new=[0, 16, 5]),
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(pool, kw, interleaved):
    kw = dict(kw)
    case(BF16, pool, kw.pop("lens"), kw.pop("t"), kw.pop("new", None), interleaved=interleaved, **kw)


@pytest.mark.parametrize("pool", BITS8)
@pytest.mark.parametrize("scale", [2.0 ** -60, 1e-4, 1.0, 3e3, 2.0 ** 90])
def test_scales_of_any_size(pool, scale):
    case(BF16, pool, [3, 16], 5, scale=scale)


@pytest.mark.parametrize("pool", [BF16, E4M3, INT8])
def test_no_check_no_query_no_rotation(pool):
    torch.manual_seed(7)
    cache = make_cache(pool, [4, 30], 8)
    k, v = (torch.randn(2, 2, 8, 64, device=DEV).to(BF16) for _ in range(2))
    before = snapshot(cache)
    out = ax.append_tokens(cache, k, v, check=False)
    assert out.seq_lengths.tolist() == [12, 38]
    z = 0 * k.double()
    check_pools(out, before, {"key": (k.double(), z), "value": (v.double(), z)}, [4, 30], [8, 8], pool)


@pytest.mark.parametrize("pool", BITS8)
def test_zero_tokens_give_the_least_scale(pool):
    cache = make_cache(pool, [0], 16)
    z = torch.zeros(1, 2, 3, 64, device=DEV, dtype=BF16)
    out = ax.append_tokens(cache, z, z)
    page = int(out.block_table[0, 0])
    assert bool((out.key_scales[page] == 2.0 ** -100).all())
    k, v = ax.gather_tokens(out, None, 4)
    assert bool((k == 0).all()) and bool((v == 0).all())
    # and a later token sets the scale
    one = torch.ones(1, 2, 1, 64, device=DEV, dtype=BF16)
    out = ax.append_tokens(out, one, one)
    k, v = ax.gather_tokens(out, None, 4)
    assert bool((k[:, :, :3] == 0).all()) and bool((k[:, :, 3] == 1).all()) and bool((v[:, :, 3] == 1).all())


@pytest.mark.parametrize("pool", BITS8)
@pytest.mark.parametrize("edge", [448.0, 127.0, 448.5, 127.5, 2.0 ** 127, 3.38e38])
def test_borders_of_the_scale(pool, edge):
    most = 448.0 if pool == E4M3 else 127.0
    x = torch.zeros(1, 2, 2, 64, device=DEV)
    x[..., 3] = edge
    cache = make_cache(pool, [0], 16)
    out = ax.append_tokens(cache, x, -x)
    s = float(out.key_scales[int(out.block_table[0, 0]), 0])
    top = 448.0 * 2.0 ** 119 if pool == E4M3 else 127.0 * 2.0 ** 121  # what fp32 holds of code * scale
    edge = min(edge, top)
    assert math.log2(s).is_integer() and most * s >= edge > most * s / 2
    k, v = ax.gather_tokens(out, None, 2, dtype=F32)
    half = 2.0 ** -4 * edge if pool == E4M3 else s / 2
    assert abs(float(k[0, 0, 0, 3]) - edge) <= half and torch.equal(k, -v)


def test_one_token_after_another_equals_exact_codes_when_scales_stay():
    """Tokens one by one: with a first token that sets the scale, the codes are those of one call."""
    torch.manual_seed(8)
    x = torch.randn(1, 2, 16, 64, device=DEV).clamp(-3.5, 3.5)
    x[:, :, 0, 0] = 4.0
    for pool in BITS8:
        a, b = make_cache(pool, [0], 16, seed=1), make_cache(pool, [0], 16, seed=1)
        a = ax.append_tokens(a, x, x)
        for i in range(16):
            b = ax.append_tokens(b, x[:, :, i:i + 1], x[:, :, i:i + 1], check=False)
        assert torch.equal(as_bytes(a.key_pool), as_bytes(b.key_pool))
        assert torch.equal(a.key_scales, b.key_scales) and torch.equal(a.seq_lengths, b.seq_lengths)


def test_e4m3_codes_keep_their_values_when_the_scale_grows():
    torch.manual_seed(9)
    x = torch.randn(1, 2, 9, 64, device=DEV)
    cache = ax.append_tokens(make_cache(E4M3, [0], 16), x, x)
    k0, _ = ax.gather_tokens(cache, None, 9, dtype=F32)
    big = torch.full((1, 2, 1, 64), 1000.0, device=DEV)
    cache = ax.append_tokens(cache, big, big)
    k1, _ = ax.gather_tokens(cache, None, 9, dtype=F32)
    normal = k0.abs() >= 2.0 ** -6 * float(cache.key_scales.max())
    assert torch.equal(k0[normal], k1[normal])
    assert float((k0 - k1).abs().max()) <= 2.0 ** -10 * 4.0  # (the scale is 4: 1000 <= 448 * 4)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_not_finite(bad):
    x = torch.ones(1, 2, 3, 64, device=DEV)
    x[0, 0, 1, 5] = bad
    # e4m3: that value alone; the scale goes by the others
    out = ax.append_tokens(make_cache(E4M3, [0], 16), x, x)
    k, v = ax.gather_tokens(out, None, 3)
    assert bool(torch.isnan(k[0, 0, 1, 5])) and int(torch.isnan(k).sum()) == 1 and int(torch.isnan(v).sum()) == 1
    k[0, 0, 1, 5] = 1
    assert bool((k == 1).all())
    # int8: the page of that head, until it is begun anew
    cache = make_cache(INT8, [0], 16)
    out = ax.append_tokens(cache, x, x)
    k, _ = ax.gather_tokens(out, None, 3)
    assert bool(torch.isnan(k[0, 0]).all()) and bool((k[0, 1] == 1).all())
    one = torch.ones(1, 2, 1, 64, device=DEV)
    k, _ = ax.gather_tokens(ax.append_tokens(out, one, one), None, 4)
    assert bool(torch.isnan(k[0, 0]).all()) and bool((k[0, 1] == 1).all())
    k, _ = ax.gather_tokens(ax.append_tokens(cache, one, one), None, 1)
    assert bool((k == 1).all())


@pytest.mark.parametrize("pool", BITS8)
def test_a_nan_scale_stays_until_the_page_is_begun_anew(pool):
    cache = make_cache(pool, [5], 16)
    page = int(cache.block_table[0, 0])
    cache.value_scales[page, 1] = math.nan
    one = torch.ones(1, 2, 1, 64, device=DEV)
    out = ax.append_tokens(cache, one, one)
    assert bool(torch.isnan(out.value_scales[page, 1])) and bool(torch.isfinite(out.value_scales[page, 0]))
    new = dataclasses.replace(out, seq_lengths=torch.zeros_like(out.seq_lengths))
    assert bool(torch.isfinite(ax.append_tokens(new, one, one).value_scales[page]).all())


@pytest.mark.parametrize("pool", [BF16, E4M3, INT8])
def test_bad_pages_and_counts(pool):
    torch.manual_seed(10)
    k, v = (torch.randn(4, 2, 20, 64, device=DEV).to(BF16) for _ in range(2))
    for what in ("unallocated", "past the pool", "past the row", "count", "negative count"):
        cache = make_cache(pool, [10, 10, 10, 10], 20)
        nl = torch.tensor([20, 20, 20, 20], dtype=torch.int32, device=DEV)
        if what == "unallocated":
            cache.block_table[2, 1] = -1
        elif what == "past the pool":
            cache.block_table[2, 1] = cache.num_blocks
        elif what == "past the row":
            cache.seq_lengths[2] = 25
        else:
            nl[2] = 21 if what == "count" else -1
        before = snapshot(cache)
        with pytest.raises(ValueError, match="sequence 2"):
            ax.append_tokens(cache, k, v, new_lengths=nl)
        assert torch.equal(as_bytes(cache.key_pool), as_bytes(before["key_pool"]))
        _lib.device_status()
        out = ax.append_tokens(cache, k, v, new_lengths=nl, check=False)
        assert _lib.device_status() == _lib.NOTICE_PAGE_LIST
        assert out.seq_lengths.tolist()[2] == {"past the row": 45, "negative count": 10}.get(what, 30)
        got, _ = ax.gather_tokens(dataclasses.replace(out, seq_lengths=out.seq_lengths.clamp(max=32)), None, 30)
        for i in (0, 1, 3):  # the other sequences are complete
            off = (got[i, :, 10:30].double() - k[i].double()).abs().max()
            assert float(off) <= (0.0 if pool == BF16 else 2.0 ** -4 * 4.5)


@pytest.mark.parametrize("pool", [BF16, F32, E4M3, INT8])
def test_gather(pool):
    cache = make_cache(pool, [0, 1, 37, 64], 0, hk=3, d=24, bs=16)
    cache.block_table[cache.block_table < 0] = 0
    ks = cache.key_scales if pool in BITS8 else None
    starts = torch.tensor([0, -3, 30, 60], dtype=torch.int32, device=DEV)
    for dt in (BF16, F16, F32):
        k, v = ax.gather_tokens(cache, starts, 11, dtype=dt)
        assert k.shape == v.shape == (4, 3, 11, 24) and k.dtype == dt
        for i, (s, n) in enumerate(zip(starts.tolist(), cache.seq_lengths.tolist())):
            for j in range(11):
                p = s + j
                if not 0 <= p < n:
                    assert bool((k[i, :, j] == 0).all()) and bool((v[i, :, j] == 0).all())
                    continue
                page = int(cache.block_table[i, p // 16])
                want = cache.key_pool[page, p % 16].float()
                want = (want * ks[page][:, None] if ks is not None else want).to(dt)
                assert torch.equal(k[i, :, j], want)
    assert ax.gather_tokens(cache, None, 0)[0].shape == (4, 3, 0, 24)


def test_gather_past_the_table_row():
    cache = make_cache(BF16, [16], 0)
    cache = dataclasses.replace(cache, seq_lengths=torch.tensor([20], dtype=torch.int32, device=DEV))
    _lib.device_status()
    k, _ = ax.gather_tokens(cache, None, 20)
    assert _lib.device_status() == _lib.NOTICE_TABLE_OVERRUN
    assert bool((k[:, :, 16:] == 0).all()) and bool((k[:, :, :16] != 0).any())


@pytest.mark.parametrize("how", ["offset", "head_major", "last"])
@pytest.mark.parametrize("pool", [BF16, E4M3])
def test_input_strides(pool, how):
    torch.manual_seed(11)
    base = torch.randn(2, 2, 6, 66, device=DEV).to(BF16)
    x = {"offset": base[..., 1:65], "head_major": base[..., :64],
         "last": base[..., :64].transpose(2, 3).contiguous().transpose(2, 3)}[how]
    a, b = make_cache(pool, [3, 9], 6, seed=2), make_cache(pool, [3, 9], 6, seed=2)
    plan = ax.rotary_plan(64)
    ax.append_tokens(a, x, x, rotary=plan, check=False)
    y = x.contiguous().clone()
    ax.append_tokens(b, y, y, rotary=plan, check=False)
    assert torch.equal(as_bytes(a.key_pool), as_bytes(b.key_pool)) and torch.equal(as_bytes(a.value_pool), as_bytes(b.value_pool))


@pytest.mark.parametrize("pool", [BF16, E4M3])
def test_pools_at_odd_addresses(pool):
    torch.manual_seed(12)
    x = torch.randn(2, 2, 6, 64, device=DEV).to(BF16)
    a, b = make_cache(pool, [3, 9], 6, seed=3), make_cache(pool, [3, 9], 6, seed=3)
    moved = {}
    for name in ("key_pool", "value_pool"):
        p = getattr(b, name)
        room = torch.empty(p.numel() + 1, dtype=torch.uint8 if pool == E4M3 else p.dtype, device=DEV)[1:]
        room.copy_(as_bytes(p).reshape(-1))
        moved[name] = (room.view(p.dtype) if pool == E4M3 else room).view(p.shape)
    b = dataclasses.replace(b, **moved)
    plan = ax.rotary_plan(64)
    ax.append_tokens(a, x, x, rotary=plan, check=False)
    ax.append_tokens(b, x, x, rotary=plan, check=False)
    assert torch.equal(as_bytes(a.key_pool), as_bytes(b.key_pool))
    assert torch.equal(ax.gather_tokens(a, None, 15)[0], ax.gather_tokens(b, None, 15)[0])


def test_no_tokens_and_no_sequences():
    cache = make_cache(E4M3, [3], 4)
    x = torch.zeros(1, 2, 0, 64, device=DEV, dtype=BF16)
    assert ax.append_tokens(cache, x, x) is cache
    with pytest.raises(ValueError):
        ax.append_tokens(cache, x, x, new_lengths=[1])
    none = dataclasses.replace(cache, block_table=cache.block_table[:0], seq_lengths=cache.seq_lengths[:0])
    y = torch.zeros(0, 2, 5, 64, device=DEV, dtype=BF16)
    assert ax.append_tokens(none, y, y).seq_lengths.numel() == 0
    assert ax.gather_tokens(none, None, 5)[0].shape == (0, 2, 5, 64)


@pytest.mark.parametrize("pool", [BF16, E4M3])
def test_captured_steps(pool):
    """A captured append of one token, replayed on new inputs and lengths, equals eager calls."""
    torch.manual_seed(13)
    a, b = make_cache(pool, [3, 14], 8, seed=4), make_cache(pool, [3, 14], 8, seed=4)
    plan = ax.rotary_plan(64)
    k = torch.randn(2, 2, 1, 64, device=DEV).to(BF16)
    q = torch.randn(2, 4, 1, 64, device=DEV).to(BF16)
    lens = a.seq_lengths.clone()
    live = dataclasses.replace(a, seq_lengths=lens)
    keep = as_bytes(a.key_pool).clone(), as_bytes(a.value_pool).clone()
    scales = [x.clone() for x in (a.key_scales, a.value_scales)] if pool == E4M3 else None
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ax.append_tokens(live, k, k, rotary=plan, query=q, check=False)
    torch.cuda.current_stream().wait_stream(s)
    as_bytes(a.key_pool).copy_(keep[0])
    as_bytes(a.value_pool).copy_(keep[1])
    if scales:
        a.key_scales.copy_(scales[0])
        a.value_scales.copy_(scales[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, q2 = ax.append_tokens(live, k, k, rotary=plan, query=q, check=False)
        lens.copy_(out.seq_lengths)
    for step in range(4):
        k.copy_(torch.randn(2, 2, 1, 64, device=DEV) * (step + 1))
        q.copy_(torch.randn(2, 4, 1, 64, device=DEV))
        graph.replay()
        b, want = ax.append_tokens(b, k, k, rotary=plan, query=q)
        assert torch.equal(q2, want) and torch.equal(lens, b.seq_lengths)
    assert torch.equal(as_bytes(a.key_pool), as_bytes(b.key_pool))
    if scales:
        assert torch.equal(a.key_scales, b.key_scales)
