"""sink_window_mod on the CPU: the mask it stands for, how it flattens, and what it refuses."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200._spec import band_of, build_spec, may_empty_rows


def _spec(mod, s=8):
    return build_spec(mod, None, batch=1, heads_q=2, seq_q=s, seq_kv=s, device="cpu").struct


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (5, 2), (100, 4), (2, 50)])
def test_mod_keeps_window_and_sinks(window, sinks):
    s = 13
    i = torch.arange(s)
    x = torch.randn(1, 2, s, s)
    got = ax.sink_window_mod(window, sinks)(x, torch.zeros(1, 1, 1, 1).long(), torch.zeros(1, 2, 1, 1).long(),
                                           i.view(1, 1, s, 1), i.view(1, 1, 1, s))
    for q in range(s):
        for k in range(s):
            keep = k <= q and (q - k < window or k < sinks)
            want = x[0, 0, q, k] if keep else torch.finfo(torch.float32).min
            assert got[0, 0, q, k] == want


def test_flattening():
    m = _spec(ax.sink_window_mod(4, 2))
    assert (m.has_band, m.band_lo, m.band_hi, m.num_sinks) == (1, 0, 3, 2)
    m = _spec(ax.compose_score_mods(ax.causal_mod(), ax.sink_window_mod(4, 2), ax.alibi_mod(2)))
    assert (m.band_lo, m.band_hi, m.num_sinks) == (0, 3, 2) and m.alibi_slopes
    # a plain window that is no wider leaves nothing of the sinks beyond it
    for w in (2, 4):
        m = _spec(ax.compose_score_mods(ax.sink_window_mod(4, 2), ax.sliding_window_mod(w)))
        assert (m.band_lo, m.band_hi, m.num_sinks) == (0, w - 1, 0)
    same = ax.compose_score_mods(ax.sink_window_mod(4, 2), ax.sink_window_mod(4, 2))
    assert _spec(same).num_sinks == 2
    assert _spec(ax.causal_mod()).num_sinks == 0


def test_ring_sees_a_causal_band_and_no_empty_rows():
    mod = ax.sink_window_mod(4, 2)
    lo, hi = band_of(mod)
    assert lo == 0 and hi >= 1 << 40      # a sink is kept at any distance
    assert not may_empty_rows(mod, None)


def test_refusals():
    for args in ((0, 1), (-3, 1), (4, -1)):
        with pytest.raises(ValueError):
            ax.sink_window_mod(*args)
    with pytest.raises(NotImplementedError):
        _spec(ax.compose_score_mods(ax.sink_window_mod(4, 2), ax.sink_window_mod(4, 3)))
    with pytest.raises(NotImplementedError):
        _spec(ax.compose_score_mods(ax.sink_window_mod(4, 2), ax.sliding_window_mod(9)))


def test_attention_core_refusals():
    from attnax_b200.mha import attention_core

    x = torch.zeros(1, 4, 16)
    for kw in ({"attention_sinks": 2}, {"attention_sinks": -1, "attention_window": 4}):
        with pytest.raises(ValueError):
            attention_core(x, x, x, num_heads=2, num_kv_heads=2, **kw)


def test_c_entry_refuses_sinks_without_a_band():
    import ctypes as C

    from attnax_b200 import _lib

    lib = _lib.load()
    p = _lib.FwdParams()
    p.dtype, p.batch, p.num_heads_q, p.num_heads_kv, p.seq_q, p.seq_kv, p.head_dim = _lib.ATTN_F32, 1, 1, 1, 1, 1, 64
    p.q = p.k = p.v = p.out = 16          # never read: the mask is refused first
    for sinks, band in ((4, 0), (-1, 1)):
        p.mask.num_sinks, p.mask.has_band = sinks, band
        assert lib.attn_fwd(C.byref(p), None) == _lib.ATTN_ERR_INVALID
