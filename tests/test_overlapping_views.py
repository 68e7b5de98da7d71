"""Rows that overlap in memory (unfolded or expanded views) are read as they lie; what comes back has rows of its own."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib, rotary

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def windows(b, h, s, d, step, dtype=F32, device="cpu", seed=0):
    """(b, h, s, d): window i of a head starts ``step`` channels behind window i - 1."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(b, h, d + (s - 1) * step, generator=g).to(dtype).to(device).unfold(2, d, step)


def rows_apart(x):
    """Whether no two elements share an address and a row's channels are neighbours."""
    at = torch.zeros((), dtype=torch.int64)
    for n, stride in zip(x.shape, x.stride()):
        at = at[..., None] + torch.arange(n) * stride
    return x.stride(3) == 1 and at.unique().numel() == x.numel()


@pytest.mark.parametrize("step", [1, 8, 40, 64, 100])
@pytest.mark.parametrize("b,h,s", [(2, 2, 8), (1, 1, 8), (2, 3, 65), (1, 4, 1)])
def test_layout_of_results(monkeypatch, b, h, s, step):
    """On the host alone: the kernel steps by the first three strides and takes a row's channels as neighbours."""
    monkeypatch.setattr(_lib, "run", lambda *a: None)
    plan = ax.rotary_plan(64, device="cpu")
    for x in (windows(b, h, s, 64, step), windows(b, h, s, 64, step).transpose(1, 2),
              windows(b, h, s, 64, step).expand(b, h, s, 64), windows(b, h, s, 64, step)[:, :1].expand(b, h, s, 64)):
        q, k = rotary._launch(x, x, plan.turns, False, 1.0, None, False)
        assert q.shape == k.shape == x.shape and rows_apart(q) and rows_apart(k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("step", [1, 8, 40])
def test_apply_rotary(dtype, step):
    x, plan = windows(2, 3, 9, 64, step, dtype, DEV), ax.rotary_plan(64)
    want = ax.apply_rotary(x.contiguous(), x[:, :1].contiguous(), plan)
    got = ax.apply_rotary(x, x[:, :1], plan)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    base = torch.randn(2, 3, 64 + 8 * step, device=DEV).to(dtype).requires_grad_()
    grad = torch.randn(2, 3, 9, 64, device=DEV).to(dtype)
    (got,) = torch.autograd.grad(ax.apply_rotary(base.unfold(2, 64, step), None, plan), base, grad)
    (want,) = torch.autograd.grad(ax.apply_rotary(base.unfold(2, 64, step).contiguous(), None, plan), base, grad)
    assert torch.equal(got, want)
    (wide,) = torch.autograd.grad(ax.apply_rotary(base.unfold(2, 64, step), None, plan), base,
                                  windows(2, 3, 9, 64, 4, dtype, DEV, seed=1))
    (want,) = torch.autograd.grad(ax.apply_rotary(base.unfold(2, 64, step), None, plan), base,
                                  windows(2, 3, 9, 64, 4, dtype, DEV, seed=1).contiguous())
    assert torch.equal(wide, want)


@pytest.mark.gpu
@pytest.mark.parametrize("pool", [BF16, torch.float8_e4m3fn])
def test_append_tokens(pool):
    from tests.test_append_tokens_gpu import as_bytes, make_cache

    plan = ax.rotary_plan(64)
    a, b = make_cache(pool, [3, 20], 9), make_cache(pool, [3, 20], 9)
    q, k, v = (windows(2, h, 9, 64, 1, BF16, DEV, seed) for h, seed in ((4, 0), (2, 1), (2, 2)))
    a, qa = ax.append_tokens(a, k, v, rotary=plan, query=q)
    b, qb = ax.append_tokens(b, k.contiguous(), v.contiguous(), rotary=plan, query=q.contiguous())
    assert torch.equal(qa, qb)
    assert all(torch.equal(as_bytes(x), as_bytes(y)) for x, y in ((a.key_pool, b.key_pool), (a.value_pool, b.value_pool)))
