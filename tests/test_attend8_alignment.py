"""attn_paged_attend8 refuses tensors that its vector accesses cannot reach, on the host (no GPU)."""

import ctypes

import pytest
import torch

from attnax_b200 import _lib


def params(rows):
    x = torch.zeros(256, dtype=torch.int64)  # (the pointers are never followed)
    at = x.data_ptr() + -x.data_ptr() % 16
    p = _lib.PagedAttend8Params()
    p.dtype, p.pool_format, p.num_seqs, p.num_heads_q, p.num_heads_kv = _lib.ATTN_BF16, _lib.POOL_E4M3, 1, rows, 1
    p.head_dim, p.seq_q, p.num_blocks, p.block_size, p.max_blocks_per_seq, p.max_context = 64, 1, 4, 16, 2, 20
    for name in ("q", "key_pool", "value_pool", "key_scales", "value_scales", "block_table", "seq_lengths", "out"):
        setattr(p, name, at)
    return p, at, x


@pytest.mark.parametrize("rows", [1, 64])  # the kernel for few rows and the one for many
@pytest.mark.parametrize("name", ["q", "key_pool", "value_pool", "out"])
@pytest.mark.parametrize("off", [2, 4, 8])
def test_tensors_off_sixteen_bytes(rows, name, off):
    p, at, _keep = params(rows)
    setattr(p, name, at + off)
    with pytest.raises(NotImplementedError):
        _lib.check(_lib.load().attn_paged_attend8(ctypes.byref(p), None), "attn_paged_attend8")


@pytest.mark.parametrize("dtype", [_lib.ATTN_F32, _lib.ATTN_BF16])
def test_workspaces_off_sixteen_bytes(dtype):
    p, at, _keep = params(64)
    p.dtype, p.max_blocks_per_seq, p.max_context = dtype, 1000, 16000
    need = _lib.load().attn_paged_attend8_workspace_size(ctypes.byref(p))
    assert need > 0
    p.workspace, p.workspace_bytes = at + 8, need
    with pytest.raises(ValueError):
        _lib.check(_lib.load().attn_paged_attend8(ctypes.byref(p), None), "attn_paged_attend8")
