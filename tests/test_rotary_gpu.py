"""Rotary positions on the GPU against 64-bit angles: values, gradients, layouts, positions, captures."""

import math

import pytest
import torch

import attnax_b200 as ax
from tests._plain64 import HALF_STEP, TINY_STEP

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def turned64(x, positions, w, interleaved, magnitude=1.0, sign=1.0):
    """(values in 64 bits, bound): x (B, H, S, D), positions (B or 1, S).

    The bound: a sine or cosine is within 6 half steps of 2^-24 of its value (argument: the fixed point, the
    conversion of the rest and two roundings, times at most pi / 4; the series; its evaluation), the magnitude adds
    one rounding and the two products another two, all relative to m (|a| + |b|); the result is rounded once.
    """
    dt, n = x.dtype, w.numel()
    x = x.detach().double()
    a = sign * positions.double()[:, None, :, None] * w.to(x.device)
    c, s = magnitude * torch.cos(a), magnitude * torch.sin(a)
    y, b32 = x.clone(), torch.zeros_like(x)
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    p, q = x[..., first], x[..., second]
    y[..., first], y[..., second] = p * c - q * s, p * s + q * c
    b32[..., first] = b32[..., second] = 10 * 2.0 ** -24 * magnitude * (p.abs() + q.abs())
    return y, b32 + HALF_STEP[dt] * (y.abs() + b32) + TINY_STEP[dt]


def check(got, want, what):
    y, bound = want
    off = (got.double() - y).abs()
    assert got.shape == y.shape and bool((off <= bound).all()), f"{what}: {float((off - bound).max()):.3e} too far"


SHAPES = [  # dtype, B, Hq, Hkv, S, D, rotary
    (BF16, 2, 4, 2, 5, 128, 128), (F16, 1, 3, 1, 37, 64, 32), (F32, 2, 2, 2, 9, 64, 64), (BF16, 3, 2, 1, 1, 80, 40),
    (F16, 1, 1, 1, 3, 6, 2), (F32, 1, 5, 3, 4, 7, 6), (BF16, 1, 8, 8, 130, 256, 128), (BF16, 2, 3, 3, 11, 96, 48),
    (F32, 1, 2, 1, 6, 20, 20),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt,b,hq,hk,s,d,r", SHAPES)
def test_values_and_gradients(dt, b, hq, hk, s, d, r, interleaved):
    torch.manual_seed(s * d + r)
    kw = {"scaling": "yarn", "factor": 4.0, "original_length": 4096} if r > 2 else {}
    w, mag = ax.rotary_frequencies(r, **kw)
    plan = ax.rotary_plan(r, interleaved=interleaved, **kw)
    q = torch.randn(b, s, hq, d, device=DEV).to(dt).transpose(1, 2).requires_grad_()
    k = torch.randn(b, s, hk, d, device=DEV).to(dt).transpose(1, 2).requires_grad_()
    pos = torch.randint(0, 100000, (b, s), device=DEV)
    q2, k2 = ax.apply_rotary(q, k, plan, positions=pos)
    assert q2.stride() == q.stride() and q2.dtype == dt
    check(q2, turned64(q, pos, w, interleaved, mag), "q")
    check(k2, turned64(k, pos, w, interleaved, mag), "k")
    gq, gk = torch.randn_like(q2), torch.randn_like(k2).expand(b, hk, s, d)
    dq, dk = torch.autograd.grad((q2, k2), (q, k), (gq, gk))
    check(dq, turned64(gq, pos, w, interleaved, mag, -1.0), "dq")
    check(dk, turned64(gk, pos, w, interleaved, mag, -1.0), "dk")


def test_gradient_against_differences():
    torch.manual_seed(0)
    plan = ax.rotary_plan(6, interleaved=True, scaling="yarn", factor=2.0, original_length=64)
    x = torch.randn(1, 2, 5, 8, device=DEV, dtype=F32).requires_grad_()
    g = torch.randn_like(x)
    dx, = torch.autograd.grad(ax.apply_rotary(x, None, plan), x, g)
    d = torch.randn_like(x)
    # linear in x: one difference with step 1 has no truncation, 30 sums of fp32 roundings of values below 8
    diff = ((ax.apply_rotary(x.detach() + d, None, plan) - ax.apply_rotary(x.detach(), None, plan)).double() * g.double()).sum()
    assert abs(float(diff - (dx.double() * d.double()).sum())) < 80 * 4 * 8 * 8 * 2.0 ** -23


@pytest.mark.parametrize("positions", ["none", "row", "shared", "int64", "int16", "negative", "far"])
def test_positions(positions):
    torch.manual_seed(1)
    b, s = 3, 7
    w, _ = ax.rotary_frequencies(16)
    plan = ax.rotary_plan(16)
    x = torch.randn(b, 2, s, 24, device=DEV, dtype=F32)
    pos = {"none": None, "row": torch.arange(5, 5 + s, device=DEV, dtype=torch.int32),
           "shared": torch.arange(5, 5 + s, device=DEV, dtype=torch.int32)[None],
           "int64": torch.randint(0, 9999, (b, s), device=DEV), "int16": torch.arange(s, device=DEV, dtype=torch.int16),
           "negative": torch.randint(-5000, 0, (b, s), device=DEV, dtype=torch.int32),
           "far": 2**31 + torch.randint(0, 9999, (b, s), device=DEV)}[positions]
    got = ax.apply_rotary(x, None, plan, positions=pos)
    at = torch.arange(s, device=DEV)[None] if pos is None else (pos[None] if pos.dim() == 1 else pos)
    if positions != "far":
        check(got, turned64(x, at, w, False), positions)
    else:  # 64-bit angles of these positions are off by 2^-21 themselves
        y, bound = turned64(x, at, w, False)
        assert bool(((got.double() - y).abs() <= bound + 2.0 ** -20 * x.double().abs().amax()).all())


def test_positions_with_strides():
    torch.manual_seed(2)
    plan, (w, _) = ax.rotary_plan(8), ax.rotary_frequencies(8)
    x = torch.randn(2, 1, 6, 8, device=DEV, dtype=BF16)
    pos = torch.randint(0, 500, (6, 2, 3), device=DEV, dtype=torch.int32)[:, :, 1].T
    check(ax.apply_rotary(x, None, plan, positions=pos), turned64(x, pos, w, False), "strided")


@pytest.mark.parametrize("how", ["offset", "last", "expanded", "heads_cut", "slice"])
def test_strides_and_alignment(how):
    torch.manual_seed(3)
    plan, (w, _) = ax.rotary_plan(32), ax.rotary_frequencies(32)
    base = torch.randn(2, 3, 5, 66, device=DEV).to(BF16)
    x = {"offset": base[..., 1:65], "last": base[..., :64].transpose(1, 3).contiguous().transpose(1, 3),
         "expanded": base[:, :1, :, :64].expand(2, 4, 5, 64), "heads_cut": base[:, 1:, :, :64],
         "slice": base[:, :, ::2, 2:]}[how]
    pos = torch.arange(x.shape[2], device=DEV)[None]
    check(ax.apply_rotary(x, None, plan), turned64(x, pos, w, False), how)


def test_inverse_brings_back_and_twice_differentiable():
    torch.manual_seed(4)
    plan = ax.rotary_plan(64)
    x = torch.randn(1, 2, 50, 64, device=DEV, dtype=F32)
    back = ax.apply_rotary(ax.apply_rotary(x, None, plan), None, plan, inverse=True)
    assert float((back - x).abs().max()) <= 2 * 10 * 2.0 ** -24 * 2 * 2 * float(x.abs().max())
    x.requires_grad_()
    g = torch.randn_like(x).requires_grad_()
    dx, = torch.autograd.grad(ax.apply_rotary(x, None, plan), x, g, create_graph=True)
    u = torch.randn_like(x)
    dg, = torch.autograd.grad(dx, g, u)  # d/dg <R^T g, u> = R u
    assert torch.equal(dg, ax.apply_rotary(u, None, plan))


def test_only_one_side_needs_a_gradient():
    plan = ax.rotary_plan(8)
    q = torch.randn(1, 2, 3, 8, device=DEV, requires_grad=True)
    k = torch.randn(1, 1, 3, 8, device=DEV)
    for a, b, leaf in ((q, k, q), (k, q, q)):
        x, y = ax.apply_rotary(a, b, plan)
        dx, = torch.autograd.grad((x.sum() + 2 * y.sum()), leaf)
        assert dx.shape == leaf.shape and bool(dx.abs().sum() > 0)
    x, y = ax.apply_rotary(q, k, plan)
    dx, = torch.autograd.grad(x.sum(), q)  # nothing comes back through y
    assert dx.shape == q.shape


def test_zero_sizes_and_special_values():
    plan = ax.rotary_plan(4)
    for shape in ((0, 2, 3, 8), (2, 0, 3, 8), (2, 2, 0, 8)):
        assert ax.apply_rotary(torch.zeros(shape, device=DEV), None, plan).shape == shape
    x = torch.zeros(1, 1, 2, 8, device=DEV)
    x[0, 0, 1, 0], x[0, 0, 1, 5], x[0, 0, 1, 6] = math.nan, math.inf, math.nan
    y = ax.apply_rotary(x, None, plan)
    assert bool(torch.isnan(y[0, 0, 1, [0, 2, 6]]).all()) and math.isinf(float(y[0, 0, 1, 5]))
    assert bool((y[0, 0, 0] == 0).all()) and bool((y[0, 0, 1, [1, 3, 4, 7]] == 0).all())


def test_side_stream_and_capture():
    torch.manual_seed(5)
    plan, (w, _) = ax.rotary_plan(64), ax.rotary_frequencies(64)
    x = torch.randn(1, 2, 33, 64, device=DEV, dtype=BF16, requires_grad=True)
    g = torch.randn_like(x)
    pos = torch.zeros(1, 33, device=DEV, dtype=torch.int32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ax.apply_rotary(x, None, plan, positions=pos)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ax.apply_rotary(x, None, plan, positions=pos)
        dx, = torch.autograd.grad(y, x, g)
    for start in (3, 70000):
        pos.copy_(torch.arange(start, start + 33, device=DEV)[None])
        graph.replay()
        torch.cuda.synchronize()
        check(y, turned64(x, pos, w, False), "captured")
        check(dx, turned64(g, pos, w, False, 1.0, -1.0), "captured gradient")
