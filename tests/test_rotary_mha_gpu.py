"""attention_core with a rotary plan: values, gradients through the rotation, cached steps."""

import pytest
import torch

import attnax_b200 as ax
from attnax_b200.mha import attention_core
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def rows(seed, b, s, heads, d):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(b, s, heads * d, generator=g, device=DEV).to(BF16)


def heads(x, n):
    b, s, f = x.shape
    return x.view(b, s, n, f // n).transpose(1, 2)


@pytest.mark.parametrize("interleaved", [False, True])
def test_values_and_gradients(interleaved):
    b, s, hq, hk, d = 2, 150, 4, 2, 64
    plan = ax.rotary_plan(32, interleaved=interleaved, scaling="yarn", factor=2.0, original_length=64)
    q, k, v = (rows(i, b, s, n, d).requires_grad_() for i, n in enumerate((hq, hk, hk)))
    out = attention_core(q, k, v, num_heads=hq, num_kv_heads=hk, rotary=plan, base_score_mod=ax.causal_mod())
    # (the same through the public pieces, which their own tests hold to 64 bits)
    qr, kr = ax.apply_rotary(heads(q, hq), heads(k, hk), plan)
    want = ax.flash_attention(qr, kr, heads(v, hk).contiguous(), score_mod=ax.causal_mod())
    want = want.transpose(1, 2).reshape(b, s, hq * d)
    assert torch.equal(out, want)
    g = torch.randn_like(out)
    got, ref = torch.autograd.grad(out, (q, k, v), g), torch.autograd.grad(want, (q, k, v), g)
    for x, y in zip(got, ref):
        assert bool((x != 0).any()) and torch.equal(x, y)  # (the backward at head dim 64 sums in a fixed order)


def test_cached_steps_equal_one_pass():
    b, s, hq, hk, d = 1, 20, 4, 2, 128
    plan = ax.rotary_plan(d)
    q, k, v = rows(0, b, s, hq, d), rows(1, b, s, hk, d), rows(2, b, s, hk, d)
    cache = ax.init_kv_layer_cache(b, hk, d, 64, BF16)
    kw = dict(num_heads=hq, num_kv_heads=hk, rotary=plan)
    _, cache = attention_core(q[:, :19], k[:, :19], v[:, :19], kv_cache=cache, base_score_mod=ax.causal_mod(), **kw)
    out, cache = attention_core(q[:, 19:], k[:, 19:], v[:, 19:], kv_cache=cache, **kw)
    assert cache.length == 20
    assert torch.equal(cache.keys[:, :, :20], ax.apply_rotary(heads(k, hk), None, plan))
    qr = ax.apply_rotary(heads(q, hq)[:, :, 19:], None, plan, positions=torch.tensor([[19]], device=DEV))
    want, bound = attention64(qr, cache.keys[:, :, :20], cache.values[:, :, :20],
                              torch.ones(1, 20, dtype=torch.bool, device=DEV))
    assert_within(heads(out, hq), want, bound, "cached step")


def test_both_ways_of_turning_are_refused():
    x = rows(0, 1, 4, 2, 64)
    with pytest.raises(ValueError):
        attention_core(x, x, x, num_heads=2, num_kv_heads=2, use_rope=True, rotary=ax.rotary_plan(64))
