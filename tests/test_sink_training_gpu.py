"""Training through windows with sinks on a contiguous cache."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200.mha import attention_core
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(seed, *shape, dt=BF):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dt)


def _keep(rows, n, window, sinks):
    """The last ``rows`` of ``n`` positions."""
    q = torch.arange(n - rows, n, device=DEV)[:, None]
    k = torch.arange(n, device=DEV)[None, :]
    return (k <= q) & ((q - k < window) | (k < sinks))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("masked", [False, True])
def test_cached_continuation_is_differentiable(dt, masked):
    """attention_core on a cache: gradients of the continuation's query, key and value, in every type."""
    b, hq, hkv, d, n, m, window, sinks = 2, 4, 2, 128, 200, 37, 64, 5
    qkv = [randn(i, b, n + m, h * d, dt=dt) for i, h in enumerate((hq, hkv, hkv))]
    do = randn(9, b, m, hq * d, dt=dt)
    kw = dict(num_heads=hq, num_kv_heads=hkv, attention_window=window, attention_sinks=sinks)
    mask = torch.ones(1, 1, m, n + m, dtype=torch.bool, device=DEV) if masked else None
    with torch.no_grad():
        _, cache = attention_core(*(t[:, :n] for t in qkv), kv_cache=ax.init_kv_layer_cache(b, hkv, d, 256, dt), **kw)
    step = [t[:, n:].clone().requires_grad_(True) for t in qkv]
    out, _ = attention_core(*step, kv_cache=cache, mask=mask, **kw)
    got = torch.autograd.grad(out, step, do)
    heads = [t.view(b, n + m, -1, d).transpose(1, 2) for t in qkv]
    dh = do.view(b, m, hq, d).transpose(1, 2)
    want, bound, grads, bounds = attention64(heads[0][:, :, n:], heads[1], heads[2], _keep(m, n + m, window, sinks), dh)
    assert_within(out.view(b, m, hq, d).transpose(1, 2), want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), got, grads, bounds):
        assert_within(g.view(b, m, -1, d).transpose(1, 2), w[:, :, -m:], bd[:, :, -m:], name)


@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (32, F32)])
def test_window_over_a_contiguous_cache_is_differentiable(d, dt):
    b, hq, hkv, n, t = 1, 4, 2, 150, 9
    cache = ax.init_kv_layer_cache(b, hkv, d, 160, dt)
    cache = ax.update_kv_layer_cache(cache, randn(1, b, hkv, n, d, dt=dt), randn(2, b, hkv, n, d, dt=dt), 0)
    q, do = randn(3, b, hq, t, d, dt=dt).requires_grad_(True), randn(4, b, hq, t, d, dt=dt)
    out = ax.kv_cache_attention(q, cache, window_size=21, num_sinks=3)
    dq, = torch.autograd.grad(out, q, do)
    want, bound, grads, bounds = attention64(q.detach(), cache.keys[:, :, :n], cache.values[:, :, :n],
                                             _keep(t, n, 21, 3), do)
    assert_within(out, want, bound, "out")
    assert_within(dq, grads[0], bounds[0], "dq")


@pytest.mark.parametrize("d,dt", [(64, F32), (128, BF)])
def test_score_mod_of_rows_in_front_of_the_cache(d, dt):
    """More rows than positions: a score_mod is given all rows, those that see nothing are zeros without a gradient."""
    b, hq, hkv, n, t = 1, 4, 2, 11, 16
    cache = ax.init_kv_layer_cache(b, hkv, d, 32, dt)
    cache = ax.update_kv_layer_cache(cache, randn(1, b, hkv, n, d, dt=dt), randn(2, b, hkv, n, d, dt=dt), 0)
    q, do = randn(3, b, hq, t, d, dt=dt).requires_grad_(True), randn(4, b, hq, t, d, dt=dt)
    bias = randn(5, b, hq, t, n, dt=dt)
    got = ax.kv_cache_attention(q, cache, window_size=6, num_sinks=2, score_mod=ax.additive_bias_mod(bias))
    dq, = torch.autograd.grad(got, q, do)
    want, bound, grads, bounds = attention64(q.detach(), cache.keys[:, :, :n], cache.values[:, :, :n],
                                             _keep(t, n, 6, 2), do, bias.double())
    first = t - n
    assert float(got[:, :, :first].detach().abs().max()) == 0.0 and float(dq[:, :, :first].abs().max()) == 0.0
    assert_within(got[:, :, first:], want[:, :, first:], bound[:, :, first:], "out")
    assert_within(dq[:, :, first:], grads[0][:, :, first:], bounds[0][:, :, first:], "dq")


@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (128, F32)])
@pytest.mark.parametrize("odd", ["q", "k", "v", "do"])
def test_training_at_odd_addresses(d, dt, odd):
    """One of the tensors starts at an address that is no multiple of 16 bytes."""
    b, hq, hkv, s, window, sinks = 1, 4, 2, 300, 40, 3
    def at(seed, h, shift):  # (contiguous, `shift` elements behind an aligned address)
        return randn(seed, b * h * s * d + 8, dt=dt)[shift:shift + b * h * s * d].view(b, h, s, d)
    t = {n: at(i, h, 1 if n == odd else 0) for i, (n, h) in enumerate((("q", hq), ("k", hkv), ("v", hkv), ("do", hq)))}
    q, k, v = (t[n].requires_grad_(True) for n in ("q", "k", "v"))
    out = ax.flash_attention(q, k, v, score_mod=ax.sink_window_mod(window, sinks))
    gs = torch.autograd.grad(out, (q, k, v), t["do"])
    want, bound, grads, bounds = attention64(q.detach(), k.detach(), v.detach(), _keep(s, s, window, sinks), t["do"])
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
        assert_within(g, w, bd, name)


def test_slopes_that_change_between_calls():
    """The kernels follow a mod's slopes: replaced, or written in place on either device."""
    hq, s, d = 4, 90, 64
    q, k, v = (randn(i, 1, hq, s, d) for i in range(3))
    mod = ax.alibi_mod(hq)
    dist = (torch.arange(s, device=DEV)[:, None] - torch.arange(s, device=DEV)[None]).abs().double()

    def check(what):
        got = ax.flash_attention(q, k, v, score_mod=ax.compose_score_mods(ax.sink_window_mod(30, 2), mod))
        bias = -mod.slopes.double().to(DEV)[None, :, None, None] * dist
        want, bound = attention64(q, k, v, _keep(s, s, 30, 2), None, bias)
        assert_within(got, want, bound, what)

    check("as made")
    mod.slopes = mod.slopes * 3
    check("replaced")
    mod.slopes *= 0.1
    check("written in place")
    mod.slopes = mod.slopes.to(DEV)
    check("on the device")
    mod.slopes.mul_(5)
    check("written in place on the device")


@pytest.mark.parametrize("window", [None, 21])
def test_first_use_of_a_cache_shape_inside_a_capture(window):
    """What a capture makes is written when it is replayed: an eager call of the same shape has to make its own."""
    b, hq, hkv, n, d, max_len = 3, 4, 2, 117, 128, 336   # (a shape that no other test uses)
    cache = ax.init_kv_layer_cache(b, hkv, d, max_len, BF)
    cache = ax.update_kv_layer_cache(cache, randn(1, b, hkv, n, d), randn(2, b, hkv, n, d), 0)
    q = randn(3, b, hq, 1, d)
    kw = {} if window is None else dict(window_size=window, num_sinks=3)
    cache = ax.KVLayerCache(cache.keys, cache.values, n - (window or 0))
    n = cache.length
    warm = ax.init_kv_layer_cache(1, hkv, d, 16, BF)
    ax.kv_cache_attention(q[:1], ax.KVLayerCache(warm.keys, warm.values, 5), **kw)   # loads the kernels
    torch.cuda.synchronize()
    from attnax_b200 import kv_cache
    kv_cache._tables.clear()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = ax.kv_cache_attention(q, cache, **kw)
    eager = ax.kv_cache_attention(q, cache, **kw)
    want, bound = attention64(q, cache.keys[:, :, :n], cache.values[:, :, :n], _keep(1, n, window or n, 3))
    assert_within(eager, want, bound, "eager")
    g.replay()
    assert_within(captured, want, bound, "replayed")
