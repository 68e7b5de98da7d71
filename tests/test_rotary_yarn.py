"""The 'yarn' frequencies at the ends of their arguments (no GPU)."""

import math

import pytest
import torch

import attnax_b200 as ax


@pytest.mark.parametrize("factor", [0.25, 0.5, 1.0])
def test_magnitude_of_factors_up_to_one(factor):
    """The method scales attention by 0.1 ln(factor) + 1 where a context is stretched, and not at all elsewhere."""
    _, m = ax.rotary_frequencies(64, scaling="yarn", factor=factor, original_length=4096)
    assert m == 1.0
    assert ax.rotary_plan(64, scaling="yarn", factor=factor, original_length=4096, device="cpu").magnitude == 1.0


@pytest.mark.parametrize("factor", [1.0001, 2.0, 40.0])
def test_magnitude_of_larger_factors(factor):
    _, m = ax.rotary_frequencies(64, scaling="yarn", factor=factor, original_length=4096)
    assert m == pytest.approx(0.1 * math.log(factor) + 1, abs=1e-15)
