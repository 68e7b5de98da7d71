"""sink_window_mod on the flash kernels: forward and gradients against the formula in 64 bits."""

import math

import numpy as np
import pytest
import torch

import attnax_b200 as ax
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _keep(sq, skv, window, sinks, q_off=0, kv_off=0):
    q = torch.arange(sq, device=DEV)[:, None] + q_off
    k = torch.arange(skv, device=DEV)[None, :] + kv_off
    return (k <= q) & ((q - k < window) | (k < sinks))


def _inputs(seed, b, hq, hkv, sq, skv, d, dt):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g, device=DEV).to(dt)  # noqa: E731
    return mk(b, hq, sq, d), mk(b, hkv, skv, d), mk(b, hkv, skv, d), mk(b, hq, sq, d)


def _run(q, k, v, do, mod, mask=None):
    q, k, v = (t.clone().requires_grad_(True) for t in (q, k, v))
    out = ax.flash_attention(q, k, v, score_mod=mod, mask=mask)
    return (out, *torch.autograd.grad(out, (q, k, v), do))


BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
CASES = [
    # b, hq, hkv, s, d, dtype, window, sinks
    (1, 4, 2, 700, 128, BF, 130, 4),       # the sinks' tile apart from the window's
    (2, 4, 4, 513, 128, HF, 64, 1),        # odd length
    (1, 2, 1, 1100, 128, BF, 257, 131),    # sinks over more than one tile
    (1, 6, 2, 640, 64, BF, 100, 4),        # two-kernel backward
    (2, 4, 1, 777, 64, HF, 300, 17),
    (1, 2, 2, 1500, 128, BF, 1, 1),        # every row keeps itself and token 0
    (1, 2, 1, 300, 128, BF, 4096, 4),      # window longer than the sequence
    (1, 2, 1, 400, 128, BF, 60, 1000),     # more sinks than tokens: plain causal
    (1, 2, 2, 100, 128, BF, 20, 3),        # one-tile forward
    (1, 2, 1, 127, 64, HF, 33, 2),
    (1, 2, 1, 1, 128, BF, 5, 2),           # one token
    (1, 4, 1, 6001, 128, BF, 64, 4),       # the sinks' gradient split over several CTAs
    (1, 2, 2, 6001, 64, HF, 30, 300),
    (2, 4, 2, 200, 64, F32, 33, 4),        # 32-bit path, register tiles
    (1, 6, 1, 321, 128, F32, 100, 70),
    (2, 3, 3, 65, 128, F32, 64, 1),
    (1, 4, 2, 1030, 64, F32, 200, 131),
    (1, 2, 2, 1, 128, F32, 1, 1),
    (1, 2, 1, 150, 32, BF, 17, 5),         # head dims of the CUDA-core path
    (1, 2, 1, 90, 8, F32, 7, 40),
]


@pytest.mark.parametrize("b,hq,hkv,s,d,dt,window,sinks", CASES)
def test_forward_and_gradients(b, hq, hkv, s, d, dt, window, sinks):
    q, k, v, do = _inputs(s + window, b, hq, hkv, s, s, d, dt)
    out, dq, dk, dv = _run(q, k, v, do, ax.sink_window_mod(window, sinks))
    want, bound, grads, bounds = attention64(q, k, v, _keep(s, s, window, sinks), do)
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), (dq, dk, dv), grads, bounds):
        assert_within(g, w, bd, name)


@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (64, F32)])
def test_with_alibi_and_documents(d, dt):
    b, hq, hkv, s, window, sinks = 2, 4, 2, 600, 90, 5
    q, k, v, do = _inputs(11, b, hq, hkv, s, s, d, dt)
    docs = torch.cat([torch.zeros(b, 250), torch.ones(b, 350)], 1).to(torch.int32)
    keep = _keep(s, s, window, sinks) & (docs[:, None, :, None] == docs[:, None, None, :]).to(DEV)
    dist = (torch.arange(s, device=DEV)[:, None] - torch.arange(s, device=DEV)[None]).abs().double()
    bias = -ax.alibi_slopes(hq).double().to(DEV)[None, :, None, None] * dist
    for mods, kp, bs in [((ax.alibi_mod(hq),), _keep(s, s, window, sinks), bias),
                         ((ax.document_mask_mod(docs),), keep, None)]:
        out, *gs = _run(q, k, v, do, ax.compose_score_mods(ax.sink_window_mod(window, sinks), *mods))
        want, bound, grads, bounds = attention64(q, k, v, kp, do, bs)
        assert_within(out, want, bound, "out")
        for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
            assert_within(g, w, bd, name)


def test_bias_in_32_bits():
    """An additive bias and a boolean mask on the 32-bit path."""
    b, hq, hkv, s, d, window, sinks = 1, 4, 2, 150, 64, 40, 3
    q, k, v, do = _inputs(6, b, hq, hkv, s, s, d, F32)
    bias = _inputs(7, 1, hq, 1, s, s, 8, F32)[0][..., :1] * torch.ones(1, 1, 1, s, device=DEV)
    mask = torch.rand(1, 1, s, s, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) > 0.2
    mask |= torch.eye(s, dtype=torch.bool, device=DEV)
    mod = ax.compose_score_mods(ax.sink_window_mod(window, sinks), ax.additive_bias_mod(bias))
    out, *gs = _run(q, k, v, do, mod, mask)
    want, bound, grads, bounds = attention64(q, k, v, _keep(s, s, window, sinks) & mask, do, bias.double())
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
        assert_within(g, w, bd, name)


def test_boolean_mask_and_rows_without_keys():
    """A mask on top: rows that keep nothing average all of V (the framework's rule)."""
    b, hq, hkv, s, d, window, sinks = 1, 2, 1, 400, 128, 50, 4
    q, k, v, do = _inputs(5, b, hq, hkv, s, s, d, BF)
    mask = torch.ones(1, 1, s, s, dtype=torch.bool, device=DEV)
    mask[..., 37, :] = False
    mask[..., 300:, 2] = False
    keep = _keep(s, s, window, sinks) & mask
    out, dq, dk, dv = _run(q, k, v, do, ax.sink_window_mod(window, sinks), mask)
    want, bound, grads, bounds = attention64(q, k, v, keep, do)
    mean = v.double().mean(2, keepdim=True).repeat_interleave(hq, 1)
    want[:, :, 37] = mean[:, :, 0]
    # the mean of s values summed in 32 bits, rounded once
    bound[:, :, 37] = 2.0 ** -8 * mean[:, :, 0].abs() + s * 2.0 ** -24 * v.double().abs().mean(2)
    assert_within(out, want, bound, "out")
    # its uniform row adds dO / s to every dV row (stored once more in bf16)
    add = (do[:, :, 37].double() / s).sum(1, keepdim=True)[:, :, None]
    dvw = grads[2] + add
    assert_within(dv, dvw, bounds[2] + 2.0 ** -8 * (grads[2].abs() + dvw.abs()) + 1e-6 * add.abs(), "dv")
    assert_within(dq, grads[0], bounds[0], "dq")
    assert_within(dk, grads[1], bounds[1], "dk")


@pytest.mark.parametrize("sq,skv", [(300, 700), (700, 300), (5, 900), (900, 1)])
@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (16, F32), (64, F32), (128, F32)])
def test_unequal_lengths(sq, skv, d, dt):
    """More queries than keys: late rows keep only sinks; more keys than queries: late keys get no gradient."""
    window, sinks = 40, 3
    q, k, v, do = _inputs(sq, 1, 4, 2, sq, skv, d, dt)
    out, *gs = _run(q, k, v, do, ax.sink_window_mod(window, sinks))
    want, bound, grads, bounds = attention64(q, k, v, _keep(sq, skv, window, sinks), do)
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
        assert_within(g, w, bd, name)


@pytest.mark.parametrize("q_off,kv_off", [(0, 0), (512, 0), (512, 256), (300, 300), (2, 0)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_global_offsets(q_off, kv_off, dt):
    """One chunk pair of a longer sequence (the ring's step): sinks go by global key positions."""
    from attnax_b200._spec import build_spec
    from attnax_b200.flash import bwd_raw, fwd_raw

    window, sinks, s = 200, 260, 512
    q, k, v, do = _inputs(q_off + 3, 1, 2, 1, s, s, 128, dt)
    spec = build_spec(ax.sink_window_mod(window, sinks), None, batch=1, heads_q=2, seq_q=s, seq_kv=s,
                      device=q.device, q_offset=q_off, kv_offset=kv_off)
    spec.fix_masked_rows = False
    out, lse = fwd_raw(q, k, v, spec)
    keep = _keep(s, s, window, sinks, q_off, kv_off)
    want, bound, grads, bounds = attention64(q, k, v, keep, do)
    assert_within(out, want, bound, "out")
    empty = ~keep.any(1)
    assert bool((lse[:, :, empty] == -math.inf).all()) and bool(torch.isfinite(lse[:, :, ~empty]).all())
    for name, g, w, bd in zip(("dq", "dk", "dv"), bwd_raw(q, k, v, out, lse, do, spec), grads, bounds):
        assert_within(g, w, bd, name)


def test_strided_inputs():
    """(batch, seq, heads, dim) projections seen as (batch, heads, seq, dim)."""
    b, hq, hkv, s, d = 2, 4, 2, 500, 128
    q, k, v, do = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in _inputs(9, b, hq, hkv, s, s, d, BF))
    out, *gs = _run(q, k, v, do, ax.sink_window_mod(70, 6))
    want, bound, grads, bounds = attention64(q, k, v, _keep(s, s, 70, 6), do)
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
        assert_within(g, w, bd, name)


@pytest.mark.parametrize("dt", [BF, F32])
def test_dropped_keys_may_hold_anything_large(dt):
    """Keys that no row keeps: their scores overflow nowhere and their gradient is zero."""
    s, window, sinks = 600, 50, 4
    q, k, v, do = _inputs(21, 1, 2, 1, 40, s, 128, dt)
    k[:, :, 60:], v[:, :, 60:] = 3e38, -3e38
    out, dq, dk, dv = _run(q, k, v, do, ax.sink_window_mod(window, sinks))
    k0, v0 = k[:, :, :60], v[:, :, :60]
    want, bound, grads, bounds = attention64(q, k0, v0, _keep(40, 60, window, sinks), do)
    assert_within(out, want, bound, "out")
    assert_within(dq, grads[0], bounds[0], "dq")
    assert_within(dk[:, :, :60], grads[1], bounds[1], "dk")
    assert float(dk[:, :, 60:].abs().max()) == 0.0 and float(dv[:, :, 60:].abs().max()) == 0.0


def test_gradient_against_differences():
    """dL/dq, dL/dk, dL/dv along random directions against central differences of the 64-bit formula.

    The step of 1e-4 makes the difference quotient's own error about 1e-8 of L's third derivative;
    the kernel's gradients are 32-bit ones within 1e-4 per element (the framework's bar), so the
    directional derivative is within 1e-4 * sum|u|.
    """
    s, window, sinks = 96, 20, 3
    q, k, v, do = _inputs(2, 1, 2, 1, s, s, 32, F32)
    _, *gs = _run(q, k, v, do, ax.sink_window_mod(window, sinks))
    keep = _keep(s, s, window, sinks)

    def loss(q, k, v):
        p = torch.softmax((q @ k.repeat_interleave(2, 1).transpose(-1, -2) / math.sqrt(32))
                          .masked_fill(~keep, -math.inf), -1)
        return float((p @ v.repeat_interleave(2, 1) * do.double()).sum())

    x = [t.double() for t in (q, k, v)]
    for i in range(3):
        u = torch.from_numpy(np.random.default_rng(i).standard_normal(x[i].shape)).to(DEV)
        u = u / u.abs().sum()
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + 1e-2 * u, x[i] - 1e-2 * u
        quotient = (loss(*hi) - loss(*lo)) / 2e-2
        assert abs(quotient - float((gs[i].double() * u).sum())) <= 1e-4 + 1e-6


def test_equals_plain_window_without_sinks():
    """num_sinks = 0 is sliding_window_mod, bit for bit."""
    q, k, v, do = _inputs(1, 1, 4, 2, 400, 400, 128, BF)
    a = ax.flash_attention(q, k, v, score_mod=ax.sink_window_mod(100, 0))
    b = ax.flash_attention(q, k, v, score_mod=ax.sliding_window_mod(100))
    assert torch.equal(a, b)


def test_attention_core_with_sinks_and_cache():
    """attention_core: a prefill and a cached continuation equal the formula on the whole sequence."""
    from attnax_b200.mha import attention_core

    b, hq, hkv, d, n, m, window, sinks = 2, 4, 2, 128, 300, 3, 64, 5
    g = torch.Generator(device=DEV).manual_seed(4)
    qkv = [torch.randn(b, n + m, h * d, generator=g, device=DEV).to(BF) for h in (hq, hkv, hkv)]
    cache = ax.init_kv_layer_cache(b, hkv, d, 512, BF)
    kw = dict(num_heads=hq, num_kv_heads=hkv, attention_window=window, attention_sinks=sinks)
    first, cache = attention_core(*(t[:, :n] for t in qkv), kv_cache=cache, **kw)
    second, cache = attention_core(*(t[:, n:] for t in qkv), kv_cache=cache, **kw)
    heads = [t.view(b, n + m, -1, d).transpose(1, 2) for t in qkv]
    want, bound = attention64(*heads, _keep(n + m, n + m, window, sinks))
    got = torch.cat([first, second], 1).view(b, n + m, hq, d).transpose(1, 2)
    assert_within(got, want, bound, "attention_core")


def test_two_graphs_of_a_training_step():
    """Forward and gradients captured twice, with ALiBi; replays follow the leaves.

    (No eager graph of the same leaves is alive meanwhile: PyTorch ties a leaf's node to the stream of
    the first graph that uses it, and waiting for that stream ends the capture.)"""
    b, hq, hkv, s, d, window, sinks = 1, 4, 2, 700, 128, 90, 4
    q, k, v, do = _inputs(31, b, hq, hkv, s, s, d, BF)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    mod = ax.compose_score_mods(ax.sink_window_mod(window, sinks), ax.alibi_mod(hq))
    def step():
        out = ax.flash_attention(q, k, v, score_mod=mod)
        return (out, *torch.autograd.grad(out, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    with torch.no_grad():
        new = _inputs(32, b, hq, hkv, s, s, d, BF)
        for t, x in zip((q, k, v, do), new):
            t.copy_(x)
    for g, _ in graphs:
        g.replay()
    dist = (torch.arange(s, device=DEV)[:, None] - torch.arange(s, device=DEV)[None]).abs().double()
    bias = -ax.alibi_slopes(hq).double().to(DEV)[None, :, None, None] * dist
    want, bound, grads, bounds = attention64(q.detach(), k.detach(), v.detach(), _keep(s, s, window, sinks), do, bias)
    for _, (out, *gs) in graphs:
        assert_within(out, want, bound, "out")
        for name, g, w, bd in zip(("dq", "dk", "dv"), gs, grads, bounds):
            assert_within(g, w, bd, name)
