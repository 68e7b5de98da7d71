"""Windows at global offsets (chunks of a longer sequence), with and without sinks, against the formula in 64 bits."""

import math

import pytest
import torch

import attnax_b200 as ax
from attnax_b200._spec import build_spec
from attnax_b200.flash import bwd_raw, fwd_raw
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(seed, hq, hkv, sq, skv, d, dt):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g, device=DEV).to(dt)  # noqa: E731
    return mk(1, hq, sq, d), mk(1, hkv, skv, d), mk(1, hkv, skv, d), mk(1, hq, sq, d)


def _spec(mod, hq, sq, skv, q_off, kv_off):
    spec = build_spec(mod, None, batch=1, heads_q=hq, seq_q=sq, seq_kv=skv, device=torch.device(DEV, 0),
                      q_offset=q_off, kv_offset=kv_off)
    spec.fix_masked_rows = False
    return spec


def _positions(sq, skv, q_off, kv_off):
    return torch.arange(sq, device=DEV)[:, None] + q_off, torch.arange(skv, device=DEV)[None, :] + kv_off


@pytest.mark.parametrize("d,dt", [(64, F32), (128, F32), (8, F32), (32, BF), (16, HF), (128, BF), (64, HF)])
@pytest.mark.parametrize("q_off,kv_off", [(0, -512), (-40, -512), (0, -7)])
@pytest.mark.parametrize("window", [10, 130])
def test_plain_window_over_keys_in_front_of_position_zero(d, dt, q_off, kv_off, window):
    """Without sinks no key is one, whatever its position: the band alone decides, at negative positions too."""
    hq, hkv, sq, skv = 4, 2, 150, 700
    q, k, v, do = _inputs(window, hq, hkv, sq, skv, d, dt)
    spec = _spec(ax.sliding_window_mod(window), hq, sq, skv, q_off, kv_off)
    out, lse = fwd_raw(q, k, v, spec)
    qi, ki = _positions(sq, skv, q_off, kv_off)
    keep = (ki <= qi) & (qi - ki < window)
    assert bool(keep.any(1).all())
    want, bound, grads, bounds = attention64(q, k, v, keep, do)
    assert_within(out, want, bound, "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), bwd_raw(q, k, v, out, lse, do, spec), grads, bounds):
        assert_within(g, w, bd, name)


@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (128, F32)])
@pytest.mark.parametrize("q_off,kv_off,rows", [(1024, 512, 512), (1150, 512, 512), (1150, 512, 200), (5000, 512, 700)])
@pytest.mark.parametrize("rested", [False, True])
def test_row_tiles_that_keep_no_key(d, dt, q_off, kv_off, rows, rested):
    """Chunks behind the window and without a sink: zeros and -inf, no gradients, also of the rounding rest."""
    window, sinks, skv, hq, hkv = 200, 260, 512, 4, 2
    if rested and dt == F32:
        pytest.skip("the rest is the 16-bit types'")
    q, k, v, do = _inputs(q_off, hq, hkv, rows, skv, d, dt)
    spec = _spec(ax.sink_window_mod(window, sinks), hq, rows, skv, q_off, kv_off)
    rest = torch.full_like(q, 7.0) if rested else None
    qi, ki = _positions(rows, skv, q_off, kv_off)
    keep = (ki <= qi) & ((qi - ki < window) | (ki < sinks))
    empty = ~keep.any(1)
    # 128-row tiles without any key, alone in their pair or beside a tile with keys
    tiles = torch.cat([empty, empty.new_ones(-rows % 128)]).view(-1, 128).all(1)
    assert bool(tiles.any())
    zero = tiles.repeat_interleave(128)[:rows]
    want, bound, grads, bounds = attention64(q, k, v, keep, do)
    for _ in range(20):
        out, lse = fwd_raw(q, k, v, spec, rest=rest)
        assert float(out[:, :, zero].abs().max()) == 0.0
        if rested:
            assert float(rest[:, :, zero].abs().max()) == 0.0
        assert bool((lse[:, :, empty] == -math.inf).all()) and bool(torch.isfinite(lse[:, :, ~empty]).all())
    if bool((~empty).any()):
        assert_within(out[:, :, ~empty], want[:, :, ~empty], bound[:, :, ~empty], "out")
    for name, g, w, bd in zip(("dq", "dk", "dv"), bwd_raw(q, k, v, out, lse, do, spec, rest=rest), grads, bounds):
        assert_within(g, w, bd, name)


@pytest.mark.parametrize("b,hq,hkv,s,d,dt,window,sinks", [
    (1, 18, 18, 4300, 128, BF, 64, 4200),   # sinks in more than half of the kv tiles, 594 tiles: nothing split
    (1, 17, 17, 4500, 64, HF, 700, 9000),   # every key a sink
    (1, 4, 1, 4300, 128, BF, 64, 4200),     # as many sinks on one kv head: chunks to fill the GPU
    (2, 6, 2, 2000, 64, BF, 100, 1500),     # several sink tiles, a few chunks each
])
def test_many_sinks(b, hq, hkv, s, d, dt, window, sinks):
    """However the rows behind the windows of the sinks' tiles are shared out."""
    g = torch.Generator(device=DEV).manual_seed(s)
    mk = lambda h: torch.randn(b, h, s, d, generator=g, device=DEV).to(dt)  # noqa: E731
    q, k, v, do = mk(hq).requires_grad_(True), mk(hkv).requires_grad_(True), mk(hkv).requires_grad_(True), mk(hq)
    out = ax.flash_attention(q, k, v, score_mod=ax.sink_window_mod(window, sinks))
    gs = torch.autograd.grad(out, (q, k, v), do)
    qi, ki = _positions(s, s, 0, 0)
    keep = (ki <= qi) & ((qi - ki < window) | (ki < sinks))
    grp = hq // hkv
    for x in range(b):
        for h in range(hkv):  # one kv head at a time: the 64-bit scores of all take too much memory
            qs, ks = slice(h * grp, (h + 1) * grp), slice(h, h + 1)
            want, bound, grads, bounds = attention64(q.detach()[x:x + 1, qs], k.detach()[x:x + 1, ks],
                                                     v.detach()[x:x + 1, ks], keep, do[x:x + 1, qs])
            assert_within(out[x:x + 1, qs], want, bound, "out")
            for name, y, w, bd, hs in zip(("dq", "dk", "dv"), gs, grads, bounds, (qs, ks, ks)):
                assert_within(y[x:x + 1, hs], w, bd, name)
