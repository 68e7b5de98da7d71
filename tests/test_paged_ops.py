"""Argument checks of the window, tree and page operators, without a GPU."""

import ctypes as C

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib


def cpu_cache(**kw):
    args = dict(num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, batch_size=3, max_blocks_per_seq=4,
                device="cpu")
    args.update(kw)
    return ax.init_paged_kv_cache(**args)


Q = torch.zeros(3, 4, 2, 64, dtype=torch.bfloat16)
DRAFT = torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16)
PAR = torch.full((3, 2), -1, dtype=torch.int32)


@pytest.mark.parametrize("q", [Q[0], Q[:2], Q[:, :3], Q[..., :32]])
def test_query_shapes(q):
    with pytest.raises(ValueError):
        ax.paged_window_attention(q, cpu_cache(), window_size=4)
    with pytest.raises(ValueError):
        ax.paged_tree_attention(q, DRAFT, DRAFT, cpu_cache(), PAR)


def test_window_arguments():
    for kw in ({"window_size": 0}, {"window_size": -2}, {"window_size": 4, "num_sinks": -1}):
        with pytest.raises(ValueError):
            ax.paged_window_attention(Q, cpu_cache(), **kw)
        with pytest.raises(ValueError):
            ax.free_window(cpu_cache(), **kw)


def test_contiguous_cache_arguments():
    cache = ax.init_kv_layer_cache(1, 2, 64, 32, torch.bfloat16, device="cpu")
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    for kw in ({"num_sinks": 2}, {"window_size": 0}, {"window_size": 4, "num_sinks": -1}):
        with pytest.raises((ValueError, RuntimeError)):
            ax.kv_cache_attention(q, cache, **kw)


def test_tree_arguments():
    c = cpu_cache()
    for dk, dv in ((DRAFT[:, :1], DRAFT), (DRAFT, DRAFT[:, :, :1]), (DRAFT, None)):
        with pytest.raises(ValueError):
            ax.paged_tree_attention(Q, dk, dv, c, PAR)
    with pytest.raises(ValueError):
        ax.paged_tree_attention(Q, DRAFT, DRAFT, c, PAR[:, :1])
    with pytest.raises(ValueError):
        ax.paged_tree_attention(Q, DRAFT, DRAFT, c, PAR, tree_lengths=[1, 2])
    big = torch.zeros(3, 4, 1025, 64)
    d = torch.zeros(3, 2, 1025, 64)
    with pytest.raises(NotImplementedError):
        ax.paged_tree_attention(big, d, d, c, torch.full((3, 1025), -1))


def test_no_cpu_path():
    c = cpu_cache()
    calls = [lambda: ax.paged_window_attention(Q, c, window_size=4),
             lambda: ax.paged_tree_attention(Q, DRAFT, DRAFT, c, PAR),
             lambda: ax.copy_blocks(c, [0], [1]), lambda: ax.fork_sequences(c, [0], [1], [2]),
             lambda: ax.free_sequences(c, [0]), lambda: ax.free_window(c, window_size=3),
             lambda: ax.compact_blocks(c), lambda: ax.append_accepted(c, DRAFT, DRAFT, [[0]] * 3, [1] * 3)]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()


def test_tables_must_be_int32():
    c = cpu_cache()
    for wrong in (ax.PagedKVCache(c.key_pool, c.value_pool, c.block_table.long(), c.seq_lengths),
                  ax.PagedKVCache(c.key_pool, c.value_pool, c.block_table, c.seq_lengths.long())):
        with pytest.raises(ValueError):
            ax.paged_window_attention(Q, wrong, window_size=4)


def test_copy_lists():
    c = cpu_cache()
    for src, dst in (([0], [8]), ([-1], [1]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0.5], [1]),
                     ([[0]], [[1]]), ([1, 2], [1, 1])):
        with pytest.raises(ValueError):
            ax.copy_blocks(c, src, dst)


def test_fork_lists():
    c = cpu_cache()
    c.seq_lengths[:] = torch.tensor([17, 16, 0])
    for src, dst, free in (([3], [0], [1]), ([0], [-1], [1]), ([0, 1], [2, 2], [1, 2]), ([0], [1, 2], [1, 2]),
                           ([0], [2], [8]), ([0, 0], [1, 2], [3, 3]), ([0], [2], [])):
        with pytest.raises(ValueError):
            ax.fork_sequences(c, src, dst, free)


def test_free_lists():
    for rows in ([3], [-1], [[0]], torch.tensor([True])):
        with pytest.raises(ValueError):
            ax.free_sequences(cpu_cache(), rows)


def test_accepted_shapes():
    c = cpu_cache()
    acc = torch.zeros(3, 2, dtype=torch.int32)
    for dk, dv, a, n in ((DRAFT[:2], DRAFT[:2], acc, [1] * 3), (DRAFT, DRAFT[:, :, :1], acc, [1] * 3),
                         (DRAFT[..., :32], DRAFT[..., :32], acc, [1] * 3), (DRAFT, DRAFT, acc[:2], [1] * 3),
                         (DRAFT, DRAFT, acc[0], [1] * 3), (DRAFT, DRAFT, acc, [1] * 2)):
        with pytest.raises(ValueError):
            ax.append_accepted(c, dk, dv, a, n)


def params(**kw):
    p = _lib.PagedParams()
    p.dtype, p.num_seqs, p.num_heads_q, p.num_heads_kv, p.head_dim, p.seq_q = _lib.ATTN_BF16, 2, 4, 2, 128, 1
    p.num_blocks, p.block_size, p.max_blocks_per_seq, p.max_context = 8, 16, 4, 64
    p.q = p.key_pool = p.value_pool = p.block_table = p.seq_lengths = p.out = 16   # never followed: refused first
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,status", [
    ({"num_seqs": 0}, _lib.ATTN_ERR_INVALID), ({"num_heads_q": 3}, _lib.ATTN_ERR_INVALID),
    ({"seq_q": 0}, _lib.ATTN_ERR_INVALID), ({"q": None}, _lib.ATTN_ERR_INVALID), ({"out": 8}, _lib.ATTN_ERR_INVALID),
    ({"max_context": -1}, _lib.ATTN_ERR_INVALID), ({"dtype": _lib.ATTN_F32}, _lib.ATTN_ERR_UNSUPPORTED),
    ({"head_dim": 32}, _lib.ATTN_ERR_UNSUPPORTED), ({"block_size": 24}, _lib.ATTN_ERR_UNSUPPORTED),
    ({"num_blocks": 1 << 30}, _lib.ATTN_ERR_UNSUPPORTED), ({"max_context": 1 << 20}, _lib.ATTN_ERR_WORKSPACE),
])
def test_c_entries_refuse(kw, status):
    lib = _lib.load()
    p = params(**kw)
    assert lib.attn_paged_window(C.byref(p), 1 << 20, 4, None) == status
    t = _lib.PagedTree()
    t.draft_keys = t.draft_values = t.parents = 16
    assert lib.attn_paged_tree(C.byref(p), C.byref(t), None) == status


def test_c_entries_refuse_windows_trees_and_lists():
    lib = _lib.load()
    p = params()
    for w, s in ((0, 0), (-1, 0), (4, -1)):
        assert lib.attn_paged_window(C.byref(p), w, s, None) == _lib.ATTN_ERR_INVALID
        assert lib.attn_paged_window_workspace_size(C.byref(p), w, s) == 0
    t = _lib.PagedTree()
    assert lib.attn_paged_tree(C.byref(p), None, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_tree(C.byref(p), C.byref(t), None) == _lib.ATTN_ERR_INVALID
    t.draft_keys = t.draft_values = t.parents = 16
    t.draft_values = 24
    assert lib.attn_paged_tree(C.byref(p), C.byref(t), None) == _lib.ATTN_ERR_INVALID
    t.draft_values = 16
    p.seq_q = 1025
    assert lib.attn_paged_tree(C.byref(p), C.byref(t), None) == _lib.ATTN_ERR_UNSUPPORTED
    c = _lib.PagedCacheParams()
    assert lib.attn_paged_copy(C.byref(c), 16, 16, 1, None) == _lib.ATTN_ERR_INVALID
    c.dtype, c.num_blocks, c.block_size, c.num_heads_kv, c.head_dim = _lib.ATTN_BF16, 8, 16, 1, 64
    c.key_pool = c.value_pool = 16
    assert lib.attn_paged_copy(C.byref(c), None, 16, 1, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_copy(C.byref(c), 16, 16, -1, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_copy(C.byref(c), None, None, 0, None) == _lib.ATTN_OK
    # no tables
    assert lib.attn_paged_fork(C.byref(c), 16, 16, 1, 16, 1, 16, 16, 16, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_free(C.byref(c), 16, 1, 16, 16, 16, 16, 16, 1024, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_compact(C.byref(c), 16, 16, 16, 1024, None) == _lib.ATTN_ERR_INVALID
    c.num_seqs, c.max_blocks_per_seq, c.block_table, c.seq_lengths = 1, 1, 16, 32
    # the new table may not be the old one; scratch is the caller's
    assert lib.attn_paged_fork(C.byref(c), 16, 16, 1, 16, 1, 16, 48, 16, None) == _lib.ATTN_ERR_INVALID
    c.num_blocks = 1 << 20
    assert lib.attn_paged_free(C.byref(c), 16, 1, 48, 48, 48, 48, None, 0, None) == _lib.ATTN_ERR_WORKSPACE
    c.num_blocks = 8
    assert lib.attn_paged_free_window(C.byref(c), 0, 0, 48, 48, 48, 16, 1024, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_compact(C.byref(c), 48, 48, None, 0, None) == _lib.ATTN_ERR_WORKSPACE
    s = (C.c_int64 * 3)(64, 64, 64)
    assert lib.attn_paged_accept(C.byref(c), 16, 16, s, s, 0, 16, 1, 16, 16, None, None) == _lib.ATTN_ERR_INVALID
    assert lib.attn_paged_accept(C.byref(c), 16, 16, s, s, 4, 16, 1, 16, None, None, None) == _lib.ATTN_ERR_INVALID


def test_new_layouts_match_the_c_compiler(tmp_path):
    import pathlib
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"attn_paged_tree_t": _lib.PagedTree, "attn_paged_cache_t": _lib.PagedCacheParams}
    body = "".join(f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for c, s in structs.items() for f, _ in s._fields_)
    body += "".join(f'printf("{c} %zu\\n", sizeof({c}));' for c in structs)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{root}/include/attnb200.h"\n'
                   f"int main(void) {{ {body} return 0; }}")
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(src)], check=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    for c, s in structs.items():
        assert int(got[c]) == C.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(s, f).offset, f
