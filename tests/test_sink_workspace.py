"""How much scratch the backward with sinks asks for: a few rows per key at most, however many keys are sinks."""

import ctypes as C

import pytest

from attnax_b200 import _lib


def _bytes(b, hq, hkv, s, d, window, sinks):
    p = _lib.BwdParams()
    p.dtype, p.batch, p.num_heads_q, p.num_heads_kv, p.seq_q, p.seq_kv, p.head_dim = _lib.ATTN_BF16, b, hq, hkv, s, s, d
    for name, heads in (("q", hq), ("k", hkv), ("v", hkv), ("o", hq), ("do", hq), ("dq", hq), ("dk", hkv), ("dv", hkv)):
        setattr(p, name + "_strides", (C.c_int64 * 3)(heads * s * d, s * d, d))
    p.mask.has_band, p.mask.band_lo, p.mask.band_hi, p.mask.num_sinks = 1, 0, window - 1, sinks
    return _lib.load().attn_bwd_workspace_size(C.byref(p))


@pytest.mark.parametrize("b,hq,hkv,s,d", [(1, 32, 8, 32768, 128), (1, 32, 8, 131072, 128), (2, 16, 4, 16384, 128),
                                          (3, 12, 4, 1999, 64), (1, 8, 1, 8192, 128), (8, 64, 8, 8192, 64),
                                          (1, 1, 1, 131072, 64)])
@pytest.mark.parametrize("window", [1, 512, 4096])
def test_sinks_take_a_bounded_workspace(b, hq, hkv, s, d, window):
    """The partials: the sinks' rows once, and behind the window no more rows than dK/dV have (or 8192 per kv head,
    or 128 for each of four waves of CTAs and one of rounding up per sink tile), fp32, dV and dK."""
    plain = _bytes(b, hq, hkv, s, d, window, 0)
    last = 0
    for sinks in (1, 16, 128, 129, 1000, 4096, s // 4, s // 2, s - 1, s, 10 * s):
        rows = min(sinks, s)
        heads = b * hkv
        tiles = -(-rows // 128)
        behind = max(heads * max(s + 127, 8192), 128 * (4 * 148 + heads * tiles if heads * tiles < 4 * 148 else 0))
        extra = _bytes(b, hq, hkv, s, d, window, sinks) - plain
        assert 0 <= extra <= (heads * rows + behind) * 2 * d * 4 + 256, (sinks, extra)
        last = extra
    if b * hkv * -(-s // 128) >= 4 * 148 and s > 8192:
        assert last == 0    # every key a sink: causal attention, and no partials
