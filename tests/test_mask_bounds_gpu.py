"""Document ids, boolean masks and biases that end with their allocation: rows past the last one read none of them."""

import pytest
import torch

import attnax_b200 as ax
from tests._plain64 import assert_within, attention64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _at_the_end(x):
    """``x`` as the last bytes of a device allocation of its own."""
    torch.cuda.empty_cache()
    buf = torch.empty(24 << 20, dtype=torch.uint8, device=DEV)
    flat = buf[buf.numel() - x.numel() * x.element_size():].view(x.dtype)
    flat.copy_(x.flatten())
    return flat.view(x.shape)


@pytest.mark.parametrize("d,dt", [(128, BF), (64, HF), (128, F32), (64, F32), (32, BF), (8, F32)])
@pytest.mark.parametrize("sq,skv", [(1, 51), (13, 13), (100, 37), (130, 300), (411, 259)])
@pytest.mark.parametrize("what", ["documents", "mask", "bias", "bias 16"])
@pytest.mark.parametrize("sinks", [0, 3])
def test_nothing_is_read_past_the_end(d, dt, sq, skv, what, sinks):
    b, hq, hkv, window = 2, 4, 2, 90
    g = torch.Generator(device=DEV).manual_seed(sq + d)
    mk = lambda *s: torch.randn(s, generator=g, device=DEV).to(dt)  # noqa: E731
    q, k, v, do = mk(b, hq, sq, d), mk(b, hkv, skv, d), mk(b, hkv, skv, d), mk(b, hq, sq, d)
    qi, ki = torch.arange(sq, device=DEV)[:, None], torch.arange(skv, device=DEV)[None]
    keep = ((ki <= qi) & ((qi - ki < window) | (ki < sinks)))[None, None]
    mods, mask, bias = [ax.sink_window_mod(window, sinks)], None, None
    if what == "documents":
        n = max(sq, skv)
        ids = _at_the_end((torch.arange(n, device=DEV)[None] * 3 // n).repeat(b, 1).to(torch.int32))
        mods.append(ax.document_mask_mod(ids))
        keep = keep & (ids[:, None, :sq, None] == ids[:, None, None, :skv])
    elif what == "mask":
        mask = torch.rand(b, hq, sq, skv, generator=g, device=DEV) < 0.7
        mask[..., 0] = True
        mask = _at_the_end(mask)
        keep = keep & mask
    else:
        x = torch.randn(b, hq, sq, skv, generator=g, device=DEV)
        bias = _at_the_end(x if what == "bias" else x.to(BF))
        mods.append(ax.additive_bias_mod(bias))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = ax.flash_attention(q, k, v, score_mod=ax.compose_score_mods(*mods), mask=mask)
    gs = torch.autograd.grad(out, (q, k, v), do)
    want, bound, grads, bounds = attention64(q.detach(), k.detach(), v.detach(), keep, do,
                                             None if bias is None else bias.double())
    # (rows that keep nothing average all of V, by the framework's rule: their own test is elsewhere)
    seen = keep.expand(b, hq, sq, skv).any(-1)
    assert_within(out[seen], want[seen], bound.expand_as(want)[seen], "out")
    assert_within(gs[0], grads[0], bounds[0], "dq")
    assert_within(gs[1], grads[1], bounds[1], "dk")
    if bool(seen.all()):
        assert_within(gs[2], grads[2], bounds[2], "dv")
