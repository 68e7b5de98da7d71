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


def test_c_entries_refuse_workspaces_off_their_alignment():
    """Before anything is launched (and before their size is looked at)."""
    lib = _lib.load()
    p = _lib.PagedParams()
    p.dtype, p.num_seqs, p.num_heads_q, p.num_heads_kv, p.head_dim, p.seq_q = _lib.ATTN_BF16, 2, 4, 2, 128, 1
    p.num_blocks, p.block_size, p.max_blocks_per_seq, p.max_context = 8, 16, 4096, 65536
    p.q = p.key_pool = p.value_pool = p.block_table = p.seq_lengths = p.out = 16    # never followed
    t = _lib.PagedTree()
    t.draft_keys = t.draft_values = t.parents = 16
    for at, status in ((24, _lib.ATTN_ERR_INVALID), (32, _lib.ATTN_ERR_WORKSPACE)):
        p.workspace, p.workspace_bytes = at, 64
        assert lib.attn_paged_window_workspace_size(C.byref(p), 1 << 20, 0) > 64
        assert lib.attn_paged_window(C.byref(p), 1 << 20, 0, None) == status
        assert lib.attn_paged_tree(C.byref(p), C.byref(t), None) == status
    for dtype, d in ((_lib.ATTN_BF16, 128), (_lib.ATTN_F16, 64), (_lib.ATTN_F32, 128)):
        b = _lib.BwdParams()
        b.dtype, b.batch, b.num_heads_q, b.num_heads_kv, b.seq_q, b.seq_kv, b.head_dim = dtype, 1, 2, 1, 200, 200, d
        for name in ("q", "k", "v", "out", "d_out", "dq", "dk", "dv", "lse"):
            setattr(b, name, 16)
        for name in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
            setattr(b, name + "_strides", (C.c_int64 * 3)(400 * d, 200 * d, d))
        b.mask.has_band, b.mask.band_hi, b.mask.num_sinks = 1, 30, 4
        for at, status in ((24, _lib.ATTN_ERR_INVALID), (32, _lib.ATTN_ERR_WORKSPACE)):
            b.workspace, b.workspace_bytes = at, 64
            assert lib.attn_bwd(C.byref(b), None) == status
    c = _lib.PagedCacheParams()
    c.dtype, c.num_blocks, c.block_size, c.num_heads_kv, c.head_dim = _lib.ATTN_BF16, 1 << 20, 16, 1, 64
    c.key_pool = c.value_pool = c.block_table = c.seq_lengths = 16
    c.num_seqs = c.max_blocks_per_seq = 1
    for at, status in ((18, _lib.ATTN_ERR_INVALID), (20, _lib.ATTN_ERR_WORKSPACE)):
        assert lib.attn_paged_compact(C.byref(c), 48, 48, at, 64, None) == status
        assert lib.attn_paged_free(C.byref(c), 16, 1, 48, 48, 48, 48, at, 64, None) == status


@pytest.mark.parametrize("n,hq,hkv,t,ctx", [
    (1, 8, 2, 1, 2500), (64, 64, 8, 16, 32768), (8, 64, 8, 64, 8000),        # as few rows as ever
    (64, 64, 8, 1024, 131072), (8, 64, 8, 1024, 131072), (1, 64, 8, 1024, 1 << 20), (256, 64, 8, 128, 32768),
    (1000, 32, 8, 32, 65536), (65535, 8, 1, 1, 1 << 20), (1, 128, 1, 1024, 1 << 24),
])
def test_partials_of_window_and_tree_stay_small(n, hq, hkv, t, ctx):
    """However many rows and tokens: 1 GiB (four waves of CTAs with partials take less than that)."""
    lib = _lib.load()
    p = _lib.PagedParams()
    p.dtype, p.num_seqs, p.num_heads_q, p.num_heads_kv, p.head_dim, p.seq_q = _lib.ATTN_BF16, n, hq, hkv, 128, t
    p.num_blocks, p.block_size, p.max_blocks_per_seq, p.max_context = 8, 16, ctx // 16 + 1, ctx
    p.q = p.key_pool = p.value_pool = p.block_table = p.seq_lengths = p.out = 16
    assert lib.attn_paged_tree_workspace_size(C.byref(p)) <= (1 << 30) + 512
    for window in (1, 1000, ctx // 2, 2 * ctx):
        assert lib.attn_paged_window_workspace_size(C.byref(p), window, 4) <= (1 << 30) + 512
