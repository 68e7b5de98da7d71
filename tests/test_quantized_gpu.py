"""Attention over 8-bit pages against 64 bits."""

import dataclasses
import math

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib
from tests._plain64 import HALF_STEP, TINY_STEP
from tests.test_append_tokens_gpu import DEV, as_bytes, make_cache

pytestmark = pytest.mark.gpu
BF16, F16, F32, E4M3, INT8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8


def held(cache, i, name):
    """(tokens, Hkv, D) in 64 bits of sequence i."""
    n, bs = int(cache.seq_lengths[i]), cache.block_size
    pages = cache.block_table[i, :-(-n // bs)].long()
    x = as_bytes(getattr(cache, f"{name}_pool"))[pages]
    x = (x.view(E4M3) if cache.key_pool.dtype == E4M3 else x).double()
    return (x * getattr(cache, f"{name}_scales")[pages].double()[:, None, :, None]).flatten(0, 1)[:n]


def attention64(q, cache, sixteen=False):
    """(out, bound) in 64 bits.

    The bound: a score is a sum of D products in 32 bits of exact factors (an fp32 query is rounded to 11 bits
    first), so an exponent is off by dx = (D + 8) 2^-24 sum |q k| scale, and twice that with the largest one taken
    off; the base-2 exponential and scaling add 2^-20.  The weights are rounded to fp16 (2^-11; below 2^-30 of the
    largest by at most 2^-33 of it, times 448 a token), sums are in 32 bits.  The query is brought to
    [2^14, 2^15) by a power of two per row and held in fp16, whose least half step is 2^-25: a channel is off by at
    most 2^-39 of the row's largest, which moves a score by that times sum |k|.  ``sixteen``: the path through bf16
    or fp32 tensors, whose P is rounded to bf16.
    """
    b, hq, t, d = q.shape
    dt = q.dtype
    hk = cache.num_kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    w_step = 2.0 ** -8 if sixteen and dt == BF16 else 2.0 ** -11
    for i in range(b):
        n = int(cache.seq_lengths[i])
        keys, values = (held(cache, i, x).repeat_interleave(hq // hk, 1).transpose(0, 1) for x in ("key", "value"))
        for r in range(t):
            m = n - t + r + 1
            if m <= 0:
                continue
            k, v, x = keys[:, :m], values[:, :m], q[i, :, r].double()[:, :, None]
            p = torch.softmax((k @ x)[..., 0] / math.sqrt(d), -1)[:, None]
            o = (p @ v)[:, 0]
            dx = (k.abs() @ x.abs())[..., 0].amax(-1, keepdim=True) / math.sqrt(d)
            dx = dx * ((d + 8) * 2.0 ** -24 + (2.0 ** -11 if dt == F32 and not sixteen else 0))
            if not sixteen:
                dx = dx + 2.0 ** -39 * x.abs().amax(1) * k.abs().sum(-1).amax(-1, keepdim=True) / math.sqrt(d)
            largest = (p * v.abs().amax(-1)[:, None]).amax(-1)
            e = (p @ v.abs())[:, 0] * (w_step + 2 * dx + 2.0 ** -20 + n * 2.0 ** -24) + n * 2.0 ** -33 * 448 * largest
            out[i, :, r], bound[i, :, r] = o, e + HALF_STEP[dt] * (o.abs() + e) + TINY_STEP[dt]
    return out, bound


def check(got, want, what=""):
    out, bound = want
    assert got.shape == out.shape
    nan = torch.isnan(out)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN elsewhere"
    off = torch.where(nan, 0.0, (got.double() - out).abs())
    bound = torch.where(nan, 0.0, bound)
    assert bool((off <= bound).all()), f"{what}: {float((off - bound).max()):.3e} too far"


def query(cache, hq, t, dt=BF16, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    # codes of up to 120 at scales of 2^-9 .. 2^-6: keys of the order of one
    return torch.randn(cache.seq_lengths.numel(), hq, t, cache.head_dim, generator=g, device=DEV).to(dt)


CASES = [  # lens, Hq, Hkv, D, page, T
    ([1], 1, 1, 128, 16, 1), ([16, 15, 17, 0], 4, 2, 64, 16, 1), ([100, 2500], 32, 8, 128, 16, 1),
    ([33, 700, 64], 8, 1, 64, 32, 1), ([50, 3], 6, 2, 128, 48, 3), ([5, 4, 1, 0], 4, 4, 64, 16, 5),
    ([300, 77], 12, 4, 64, 32, 5), ([1000], 32, 4, 128, 64, 4), ([513, 40], 8, 8, 128, 128, 16),
    ([200, 130], 8, 2, 64, 16, 37), ([90], 16, 2, 128, 16, 64), ([5000, 2047, 2048, 2049], 8, 2, 128, 16, 1),
    ([40], 24, 2, 128, 16, 1), ([31, 62], 5, 5, 64, 256, 2),
]


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("lens,hq,hk,d,bs,t", CASES)
def test_against_64_bits(pool, lens, hq, hk, d, bs, t):
    cache = make_cache(pool, lens, 0, hk, d, bs, seed=len(lens) + d + t)
    q = query(cache, hq, t)
    want = attention64(q, cache)
    check(ax.paged_quantized_attention(q, cache), want, "lengths read")
    check(ax.paged_quantized_attention(q, cache, max_context=max(lens) + 1000), want, "bounded")


MANY = [  # many rows per kv head: the tcgen05 kernel
    ([700, 130, 5], 8, 2, 128, 16, 13), ([129, 128, 127, 0], 12, 4, 64, 32, 20), ([2500], 7, 1, 128, 64, 7),
    ([1100, 3], 40, 2, 64, 16, 9), ([300], 8, 1, 128, 16, 45), ([3000, 600], 16, 2, 128, 128, 70), ([64], 64, 1, 64, 16, 1),
]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("lens,hq,hk,d,bs,t", MANY)
def test_many_rows(pool, lens, hq, hk, d, bs, t, dt):
    assert hq // hk * t >= 49
    cache = make_cache(pool, lens, 0, hk, d, bs, seed=sum(lens) + t)
    q = query(cache, hq, t, dt)
    check(ax.paged_quantized_attention(q, cache, max_context=max(lens)), attention64(q, cache))


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("spread", [8, 40])
def test_many_rows_with_scales_that_differ(pool, spread):
    cache = make_cache(pool, [260, 40], 0, 2, 64, 16)
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    cache.value_scales.copy_(2.0 ** torch.randint(-spread, spread, cache.value_scales.shape, generator=g, device=DEV).float())
    cache.value_scales[int(cache.block_table[0, 3])] = 0
    cache.key_scales[int(cache.block_table[0, 4])] = 0
    cache.key_scales.mul_(1.37)
    q = query(cache, 8, 30) * 2
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_many_rows_with_growing_scores():
    cache = make_cache(INT8, [3000], 0, 1, 64, 16)
    table = cache.block_table[0].long()
    cache.key_scales[table, 0] = torch.linspace(2.0 ** -9, 2.0 ** -2, table.numel(), device=DEV)
    q = query(cache, 8, 9) * 3
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_many_rows_and_small_codes():
    """Subnormal codes are values as well."""
    cache = make_cache(E4M3, [200], 0, 1, 128, 16)
    for x in (cache.key_pool, cache.value_pool):
        x.copy_((torch.randint(-15, 16, x.shape, device=DEV) * 2.0 ** -9).to(E4M3))
    cache.key_scales.fill_(64.0)
    for t in (1, 64):
        q = query(cache, 2, t)
        check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


@pytest.mark.parametrize("t", [60, 130])
def test_many_rows_and_nan(t):
    for which in ("key", "value"):
        for back in (1, 50, 129, 140):
            cache = make_cache(E4M3, [150], 0, 2, 64, 16, seed=back)
            pos = 150 - back
            as_bytes(getattr(cache, f"{which}_pool"))[int(cache.block_table[0, pos // 16]), pos % 16, 1, 7] = 0x7F
            got = ax.paged_quantized_attention(query(cache, 4, t), cache)
            rows = 150 - t + torch.arange(t, device=DEV) >= pos
            nan = torch.isnan(got)
            assert not bool(nan[:, :2].any()) and not bool(nan[:, 2:, ~rows].any())
            assert bool((nan[:, 2:] if which == "key" else nan[:, 2:, :, 7])[:, :, rows].all())
            if which == "value":
                nan[..., 7] = False
                assert not bool(nan.any())


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 30.0])
def test_query_types_and_sizes(dt, size):
    cache = make_cache(E4M3, [70, 129], 0, 2, 128, 16)
    q = (query(cache, 8, 2, F32) * size).to(dt)
    got = ax.paged_quantized_attention(q, cache)
    assert got.dtype == dt
    check(got, attention64(q, cache))


@pytest.mark.parametrize("spread", [12, 40])
def test_query_of_widely_different_channels(spread):
    cache = make_cache(INT8, [70], 0, 1, 64, 16)
    q = query(cache, 2, 1, F32)
    q[..., ::7] *= 2.0 ** spread
    q[..., 1::7] *= 2.0 ** -spread
    cache.key_pool[:, :, :, ::7] = 0  # (else the scores are all of the large channels)
    check(ax.paged_quantized_attention(q.to(BF16), cache), attention64(q.to(BF16), cache))


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("spread", [8, 40])
def test_scales_that_differ_between_pages(pool, spread):
    """Values of very different sizes from page to page: the weights keep their digits."""
    cache = make_cache(pool, [260, 40], 0, 2, 64, 16)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    cache.value_scales.copy_(2.0 ** torch.randint(-spread, spread, cache.value_scales.shape, generator=g, device=DEV).float())
    q = query(cache, 4, 1) * 2
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_small_page_with_the_large_weight():
    """A page of tiny values that gets nearly all of the weight, behind one of huge values that gets none."""
    cache = make_cache(E4M3, [32], 0, 1, 64, 16)
    p0, p1 = cache.block_table[0].tolist()
    k = torch.zeros_like(cache.key_pool, dtype=F32)
    k[p0], k[p1] = -1.0, 1.0
    cache.key_pool.copy_(k.to(E4M3))
    cache.key_scales.fill_(2.0)
    cache.value_scales[p0], cache.value_scales[p1] = 2.0 ** 30, 2.0 ** -8
    q = torch.full((1, 2, 1, 64), 3.0, device=DEV, dtype=BF16)  # scores of +-48: a weight of e^-96 against 2^38
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_scales_off_powers_of_two_and_zero():
    cache = make_cache(INT8, [100], 0, 2, 128, 16)
    cache.key_scales.mul_(1.37)
    cache.value_scales.mul_(0.61)
    cache.value_scales[int(cache.block_table[0, 1])] = 0
    cache.key_scales[int(cache.block_table[0, 2])] = 0
    q = query(cache, 4, 2)
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_growing_scores_move_the_maximum():
    cache = make_cache(INT8, [4000], 0, 1, 64, 16)
    table = cache.block_table[0].long()
    cache.key_scales[table, 0] = torch.linspace(2.0 ** -9, 2.0 ** -2, table.numel(), device=DEV)
    q = query(cache, 8, 1) * 3
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_slots_behind_the_sequence_hold_anything():
    cache = make_cache(E4M3, [5, 17, 33], 0, 2, 128, 16)
    q = query(cache, 4, 2)
    want = ax.paged_quantized_attention(q, cache)
    check(want, attention64(q, cache))
    codes = as_bytes(cache.key_pool), as_bytes(cache.value_pool)
    for i, n in enumerate(cache.seq_lengths.tolist()):
        page = int(cache.block_table[i, (n - 1) // 16])
        for x in codes:
            x[page, n % 16:] = 0x7F  # NaN
    cache.block_table[0, 1:] = 10**6  # and entries behind the last page are not read
    assert torch.equal(ax.paged_quantized_attention(q, cache), want)


@pytest.mark.parametrize("t", [1, 3, 20])
def test_nan_reaches_the_rows_that_see_it(t):
    """A NaN key or value: rows at or behind it are NaN, rows in front of it are not."""
    for which in ("key", "value"):
        for back in (1, 2, t, t + 5):
            if back > 40:
                continue
            cache = make_cache(E4M3, [41], 0, 2, 64, 16, seed=back)
            pos = 41 - back
            as_bytes(getattr(cache, f"{which}_pool"))[int(cache.block_table[0, pos // 16]), pos % 16, 1, 7] = 0xFF
            q = query(cache, 4, t)
            got = ax.paged_quantized_attention(q, cache)
            rows = 41 - t + torch.arange(t, device=DEV) >= pos
            assert not bool(torch.isnan(got[:, :2]).any())
            if which == "key":
                assert torch.equal(torch.isnan(got[:, 2:]), rows[None, None, :, None].expand(1, 2, t, 64))
            else:
                assert bool(torch.isnan(got[:, 2:, :, 7])[:, :, rows].all())
                assert not bool(torch.isnan(got[:, 2:, ~rows]).any())


def test_page_with_a_nan_scale():
    cache = make_cache(INT8, [40], 0, 2, 64, 16)
    cache.value_scales[int(cache.block_table[0, 2]), 0] = math.nan  # tokens 32 .. 39
    q = query(cache, 4, 12)  # rows at 28 .. 39
    got = ax.paged_quantized_attention(q, cache)
    assert bool(torch.isnan(got[:, :2, 4:]).all()) and not bool(torch.isnan(got[:, :2, :4]).any())
    assert not bool(torch.isnan(got[:, 2:]).any())


def test_nan_and_infinite_queries_stay_in_their_row():
    cache = make_cache(E4M3, [40], 0, 2, 64, 16)
    q = query(cache, 4, 3)
    want = ax.paged_quantized_attention(q, cache)
    q[0, 1, 0, 3], q[0, 3, 2, 0] = math.nan, math.inf
    got = ax.paged_quantized_attention(q, cache)
    bad = torch.zeros(1, 4, 3, dtype=torch.bool, device=DEV)
    bad[0, 1, 0] = bad[0, 3, 2] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])


def test_rows_in_front_of_the_sequence_are_zeros():
    cache = make_cache(E4M3, [3, 0, 9], 0, 2, 128, 16)
    q = query(cache, 4, 7)
    got = ax.paged_quantized_attention(q, cache)
    assert bool((got[0, :, :4] == 0).all()) and bool((got[1] == 0).all()) and bool((got[0, :, 4:] != 0).any())
    check(got, attention64(q, cache))


def test_lengths_past_the_bound_and_the_table():
    cache = make_cache(INT8, [5000, 100], 0, 1, 64, 16)
    q = query(cache, 2, 1)
    _lib.device_status()
    got = ax.paged_quantized_attention(q, cache, max_context=2500)
    assert _lib.device_status() == _lib.NOTICE_CONTEXT_OVERRUN
    check(got[1:], tuple(x[1:] for x in attention64(q, cache)))
    got = ax.paged_quantized_attention(q, cache, max_context=40)  # one split, of 64 tokens
    assert _lib.device_status() == _lib.NOTICE_CONTEXT_OVERRUN
    many = query(cache, 64, 1)
    ax.paged_quantized_attention(many, cache, max_context=40)
    assert _lib.device_status() == _lib.NOTICE_CONTEXT_OVERRUN
    ax.paged_quantized_attention(many, cache, max_context=5000)
    assert _lib.device_status() == 0
    longer = dataclasses.replace(cache, seq_lengths=torch.tensor([6000, 100], dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        ax.paged_quantized_attention(q, longer)
    got = ax.paged_quantized_attention(q, longer, max_context=6000)
    assert _lib.device_status() == _lib.NOTICE_TABLE_OVERRUN
    full = dataclasses.replace(cache, seq_lengths=torch.tensor([cache.block_table.shape[1] * 16, 100],
                                                               dtype=torch.int32, device=DEV))
    check(got, attention64(q, full))


@pytest.mark.parametrize("d,bs,odd", [(80, 16, False), (128, 24, False), (64, 16, True), (32, 8, False)])
@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_other_caches(d, bs, odd, dt):
    cache = make_cache(E4M3, [50, 7, 0], 0, 2, d, bs)
    if odd:
        room = torch.empty(cache.key_pool.numel() + 1, dtype=torch.uint8, device=DEV)[1:]
        room.copy_(as_bytes(cache.key_pool).reshape(-1))
        cache = dataclasses.replace(cache, key_pool=room.view(E4M3).view(cache.key_pool.shape))
    q = query(cache, 4, 9, dt)
    if d == 80:  # no attention kernel of this package has that head_dim
        with pytest.raises(NotImplementedError):
            ax.paged_quantized_attention(q, cache)
        return
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache, sixteen=True))


def test_shared_pages_and_strided_queries():
    cache = make_cache(E4M3, [40, 40], 0, 2, 64, 16)
    cache.block_table[1] = cache.block_table[0]
    q = torch.randn(2, 3, 4, 64, device=DEV).to(BF16).transpose(1, 2)
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))


def test_same_result_twice_and_on_another_stream():
    cache = make_cache(E4M3, [9000, 12], 0, 2, 128, 16)
    q = query(cache, 8, 2)
    want = ax.paged_quantized_attention(q, cache)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ax.paged_quantized_attention(q, cache, max_context=9000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and torch.equal(ax.paged_quantized_attention(q, cache), want)


def test_a_decode_loop_captured():
    """Append and attend as a serving step would, captured once and replayed, against eager steps."""
    torch.manual_seed(5)
    plan = ax.rotary_plan(64)
    caches = [make_cache(E4M3, [20, 63], 8, 2, 64, 16, seed=6) for _ in range(2)]
    lens = caches[0].seq_lengths.clone()
    live = dataclasses.replace(caches[0], seq_lengths=lens)
    k, v = (torch.randn(2, 2, 1, 64, device=DEV).to(BF16) for _ in range(2))
    q = torch.randn(2, 4, 1, 64, device=DEV).to(BF16)
    ax.paged_quantized_attention(q, live, max_context=80)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, q2 = ax.append_tokens(live, k, v, rotary=plan, query=q, check=False)
        out = ax.paged_quantized_attention(q2, new, max_context=80)
        lens.copy_(new.seq_lengths)
    eager = caches[1]
    for step in range(4):
        k.copy_(torch.randn(2, 2, 1, 64, device=DEV))
        v.copy_(torch.randn(2, 2, 1, 64, device=DEV) * 2.0 ** step)
        q.copy_(torch.randn(2, 4, 1, 64, device=DEV))
        graph.replay()
        eager, qe = ax.append_tokens(eager, k, v, rotary=plan, query=q)
        want = ax.paged_quantized_attention(qe, eager, max_context=80)
        assert torch.equal(out, want)
        check(want, attention64(qe, eager))


def test_prompt_then_decode():
    """A prompt and some steps: allocated, appended to both kinds of cache, attended."""
    torch.manual_seed(6)
    hk, hq, d, n = 2, 4, 128, 50
    plan = ax.rotary_plan(d)
    q8 = ax.init_quantized_paged_kv_cache(num_blocks=8, block_size=16, num_kv_heads=hk, head_dim=d, batch_size=1,
                                          max_blocks_per_seq=4)
    wide = ax.init_paged_kv_cache(num_blocks=8, block_size=16, num_kv_heads=hk, head_dim=d, batch_size=1,
                                  max_blocks_per_seq=4)
    q8, _ = ax.allocate_blocks(q8, sequence_idx=0, num_new_tokens=n + 3, free_block_ids=[5, 1, 7, 2])
    wide, _ = ax.allocate_blocks(wide, sequence_idx=0, num_new_tokens=n + 3, free_block_ids=[5, 1, 7, 2])
    assert isinstance(q8, ax.QuantizedPagedKVCache)
    for t in (n, 1, 2):
        k, v = (torch.randn(1, hk, t, d, device=DEV).to(BF16) for _ in range(2))
        q = torch.randn(1, hq, t, d, device=DEV).to(BF16)
        q8, qa = ax.append_tokens(q8, k, v, rotary=plan, query=q)
        wide, qb = ax.append_tokens(wide, k, v, rotary=plan, query=q)
        assert torch.equal(qa, qb)
        check(ax.paged_quantized_attention(qa, q8), attention64(qa, q8))


@pytest.mark.parametrize("t", [1, 30])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_query_off_sixteen_bytes(t, dt):
    cache = make_cache(E4M3, [50, 33], 0, 2, 64, 16)
    q = query(cache, 4, t, dt)
    room = torch.empty(q.numel() + 1, dtype=dt, device=DEV)[1:]
    room.copy_(q.reshape(-1))
    odd = room.view(q.shape)
    assert odd.is_contiguous() and odd.data_ptr() % 16
    got = ax.paged_quantized_attention(odd, cache)
    assert torch.equal(got, ax.paged_quantized_attention(q, cache))
    check(got, attention64(q, cache))


def test_bounds_of_any_size():
    cache = make_cache(E4M3, [50, 0], 0, 2, 64, 16)
    q = query(cache, 4, 2)
    want = ax.paged_quantized_attention(q, cache)
    for bound in (50, 2**31, 2**40):
        assert torch.equal(ax.paged_quantized_attention(q, cache, max_context=bound), want)
    assert _lib.device_status() == 0
    zero = dataclasses.replace(cache, seq_lengths=torch.zeros_like(cache.seq_lengths))
    assert not ax.paged_quantized_attention(q, zero, max_context=0).any()


@pytest.mark.parametrize("pool", [E4M3, INT8])
@pytest.mark.parametrize("where", ["keys", "values", "both"])
@pytest.mark.parametrize("step", [4, 10])
def test_many_rows_whose_maxima_grow_within_a_tile(pool, where, step):
    """Of every 128 tokens the later 64 bring larger scores, larger values or both, more with every tile."""
    cache = make_cache(pool, [500, 300], 0, 2, 128, 16, seed=step)
    q = query(cache, 8, 40)
    for b in range(2):
        for i, page in enumerate(cache.block_table[b].tolist()):
            if page < 0:
                continue
            grow = 2.0 ** (step * (i // 8 + (i // 4) % 2))
            if where != "values":
                cache.key_scales[page] *= grow ** 0.25
            if where != "keys":
                cache.value_scales[page] *= grow
    check(ax.paged_quantized_attention(q, cache), attention64(q, cache))
