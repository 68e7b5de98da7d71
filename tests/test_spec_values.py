"""What build_spec hands to the kernels follows the mods' values, on the CPU."""

import ctypes as C

import pytest
import torch

import attnax_b200 as ax
from attnax_b200._spec import build_spec


def _spec(mod, s=8, heads=4):
    return build_spec(mod, None, batch=1, heads_q=heads, seq_q=s, seq_kv=s, device="cpu")


def _slopes(spec, n):
    return list((C.c_float * n).from_address(spec.struct.alibi_slopes))


def test_slopes_follow_the_mod():
    mod = ax.alibi_mod(4)
    assert _slopes(_spec(mod), 4) == mod.slopes.tolist()
    mod.slopes = mod.slopes * 3
    assert _slopes(_spec(mod), 4) == mod.slopes.tolist()
    mod.slopes *= 0.5
    assert _slopes(_spec(mod), 4) == mod.slopes.tolist()


def test_device_copies_follow_their_values():
    """The copy kept for a device (a stand-in here) is made again when the host's values, length or type change."""
    mod = ax.alibi_mod(4)
    one = mod._device_tensor("slopes", mod.slopes, "meta")
    assert mod._device_tensor("slopes", mod.slopes, "meta") is one
    assert mod._device_tensor("slopes", mod.slopes.clone(), "meta") is one
    mod.slopes[2] += 1
    two = mod._device_tensor("slopes", mod.slopes, "meta")
    assert two is not one and mod._device_tensor("slopes", mod.slopes, "meta") is two
    assert mod._device_tensor("slopes", mod.slopes.double(), "meta").dtype == torch.float64
    assert mod._device_tensor("slopes", mod.slopes[:3], "meta").shape == (3,)


def test_a_sink_window_without_sinks_is_a_plain_window():
    """It composes like one: with wider and narrower windows, with other windows without sinks, and with sinks."""
    def band(*mods):
        m = _spec(ax.compose_score_mods(*mods)).struct
        return m.has_band, m.band_lo, m.band_hi, m.num_sinks

    assert band(ax.sink_window_mod(4, 0), ax.sliding_window_mod(9)) == (1, 0, 3, 0)
    assert band(ax.sliding_window_mod(3, causal=False), ax.sink_window_mod(4, 0)) == (1, 0, 2, 0)
    assert band(ax.sink_window_mod(4, 0), ax.sink_window_mod(7, 0)) == (1, 0, 3, 0)
    assert band(ax.sink_window_mod(4, 0), ax.sink_window_mod(7, 2)) == (1, 0, 3, 0)
    assert band(ax.sink_window_mod(7, 2), ax.sink_window_mod(7, 0)) == (1, 0, 6, 0)
    assert band(ax.sink_window_mod(4, 0)) == (1, 0, 3, 0)
    with pytest.raises(NotImplementedError):
        band(ax.sink_window_mod(7, 2), ax.sink_window_mod(9, 0))


@pytest.mark.parametrize("window,sinks", [(1 << 70, 4), (5, (1 << 64) + 3), ((1 << 64) + 5, (1 << 64) + 3)])
def test_windows_and_sinks_beyond_64_bits(window, sinks):
    """Longer than any sequence, not their low 64 bits."""
    m = _spec(ax.sink_window_mod(window, sinks)).struct
    assert m.has_band and m.band_lo == 0
    assert m.band_hi == (window - 1 if window < 1 << 60 else m.band_hi) and m.band_hi >= min(window - 1, 1 << 60)
    assert m.num_sinks == (sinks if sinks < 1 << 60 else m.num_sinks) and m.num_sinks >= min(sinks, 1 << 60)
    # positions up to 2^40 added on either side stay within 64 bits
    assert m.band_hi + (1 << 40) < 1 << 63 and m.num_sinks + (1 << 40) < 1 << 63
