"""The 'yarn' ramp where all pairs lie on one side of it (no GPU)."""

import math

import pytest
import torch

import attnax_b200 as ax


def quotients(**kw):
    """Each pair's frequency over its plain one, and its turns within original_length."""
    w, _ = ax.rotary_frequencies(16, scaling="yarn", factor=4.0, **kw)
    plain, _ = ax.rotary_frequencies(16, base=kw.get("base", 10000.0))
    return (w / plain).tolist(), (kw["original_length"] * plain / (2 * math.pi)).tolist()


@pytest.mark.parametrize("kw", [{"original_length": 3}, {"original_length": 6},
                                {"original_length": 1000, "beta_slow": 200.0, "beta_fast": 400.0}])
def test_pairs_that_all_turn_too_rarely_are_all_stretched(kw):
    q, turns = quotients(**kw)
    assert max(turns) < kw.get("beta_slow", 1.0)
    assert q == [0.25] * 8


def test_pairs_that_all_turn_often_keep_their_frequency():
    q, turns = quotients(original_length=10**9, base=1.5)
    assert min(turns) > 32 and q == [1.0] * 8


@pytest.mark.parametrize("base", [0.5, 0.999])
def test_frequencies_that_grow_are_refused(base):
    """The ramp runs from fast pairs to slow ones: it has no meaning for a base below 1."""
    with pytest.raises(ValueError, match="base above 1"):
        ax.rotary_frequencies(16, scaling="yarn", factor=4.0, original_length=4096, base=base)
