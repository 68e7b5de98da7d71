"""Forward-mode tangents are refused where there is no formula for them, not dropped."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import attnax_b200 as ax
from attnax_b200 import rotary


def dual(x, on=True):
    return fw.make_dual(x, torch.ones_like(x)) if on else x


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["query", "key", "both"])
def test_rotary_on_the_host(monkeypatch, which, grad):
    """The launch replaced by copies: what counts is whether the autograd function sees the tangent."""
    monkeypatch.setattr(rotary, "_launch", lambda q, k, *a: (q.clone(), None if k is None else k.clone()))
    plan = ax.rotary_plan(8, device="cpu")
    how = (plan.turns, None, plan.interleaved, plan.magnitude, False)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        q, k = (dual(torch.ones(1, 2, 3, 8), which in (name, "both")) for name in ("query", "key"))
        with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|jvp"):
            rotary._turned(q, k, *how)
        with torch.no_grad():
            rotary._turned(torch.ones(1, 2, 3, 8), None, *how)  # no tangent: as ever


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_on_the_gpu(which):
    x = [torch.randn(1, 2, 8, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    plan = ax.rotary_plan(64)
    want, turned = ax.flash_attention(*x), ax.apply_rotary(x[0], x[1], plan)
    with fw.dual_level():
        d = [dual(t, i == which) for i, t in enumerate(x)]
        with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|jvp"):
            ax.flash_attention(*d)
        if which < 2:
            with pytest.raises((NotImplementedError, RuntimeError), match="forward mode|jvp"):
                ax.apply_rotary(d[0], d[1], plan)
        assert torch.equal(ax.flash_attention(*x), want)
        assert all(torch.equal(a, b) for a, b in zip(ax.apply_rotary(x[0], x[1], plan), turned))
