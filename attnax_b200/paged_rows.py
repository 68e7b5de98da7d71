"""Several query rows per sequence over the paged cache: windows with sinks and trees of drafted tokens.

``paged_window_attention`` is the decode of a model whose layers slide
(``sink_window_mod`` in training): the query rows are the last positions of
each sequence, and only the window's pages and the sinks' are read.
``paged_tree_attention`` scores a tree of drafted tokens in one pass: every
row sees the cached context and the drafts on its own path.  Both have no
counterpart in the reference, whose decode lets every row see the whole
context (attnax/kernels/paged.py:17-84).

bf16/f16 caches with head_dim 64 or 128 and a block size that is a multiple
of 16 take the fused kernels (one launch, and one that joins the splits);
other caches gather each sequence and run the flash kernel on it, waiting for
the lengths (``max_context`` is not used there).  Both kernels run on the
current stream of the cache's device.
Like the paged decode they are for inference: the fused kernels have no backward,
and what they return carries no gradient.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._spec import dtype_code
from .flash import attention, softmax_scale
from .paged import PagedKVCache, check_pools, check_rows, gather_kv, gather_positions, pools_by_tma, refuse_codes


def _check_query(query, cache: PagedKVCache):
    if not isinstance(query, torch.Tensor) or query.dim() != 4:
        raise ValueError("query must be (num_seqs, num_heads, seq_q, head_dim)")
    n, hq, t, d = query.shape
    pool, rows = check_tables(cache)
    if n != rows[0]:
        raise ValueError(f"query has {n} sequences, the cache {rows[0]}")
    if hq % pool[2] != 0:
        raise ValueError(f"num_heads ({hq}) must be divisible by num_kv_heads ({pool[2]})")
    if d != pool[3]:
        raise ValueError(f"query head_dim {d} != cache head_dim {pool[3]}")
    return n, hq, t, d, pool, rows


def check_tables(cache: PagedKVCache):
    """The kernels read int32 tables on the pools' device, a row and a length per sequence, and two pools alike.

    Returns the pools' shape and the table's.
    """
    k, v, table, lengths = cache.key_pool, cache.value_pool, cache.block_table, cache.seq_lengths
    pool, rows, dev = k.shape, table.shape, k.device
    # (one pass where all is well: these checks are a good part of a small call's host time)
    if (len(pool) == 4 and v.shape == pool and v.dtype is k.dtype and v.device == dev
            and len(rows) == 2 and lengths.shape == rows[:1] and table.dtype is torch.int32
            and lengths.dtype is torch.int32 and table.device == dev and lengths.device == dev):
        return pool, rows
    check_pools(cache)
    check_rows(table, lengths)
    for name, x in (("block_table", table), ("seq_lengths", lengths)):
        if x.device != dev:
            raise RuntimeError(f"{name} must be on the pools' device")
    return pool, rows


def narrow(x: torch.Tensor, device) -> torch.Tensor:
    """Integers as contiguous int32 on the device; what 32 bits do not hold becomes their end of the range,
    which no index reaches."""
    if x.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
        if x.is_floating_point() or x.is_complex() or x.dtype == torch.bool:
            if x.numel():
                raise ValueError(f"indices and lengths must be integers, got {x.dtype}")
        else:
            x = x.clamp(-2**31, 2**31 - 1)
    return x.to(device=device, dtype=torch.int32).contiguous()


def on_device(x, device) -> torch.Tensor:
    """int32, contiguous, on the device."""
    if isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.device == device:
        return x.contiguous()
    return narrow(torch.as_tensor(x), device)


def _need_cuda(query, cache: PagedKVCache):
    if not query.is_cuda or query.device != cache.key_pool.device:
        raise RuntimeError("attnax_b200 kernels need the query on the cache's CUDA device; there is no CPU path")


def _fused(cache: PagedKVCache, pool) -> bool:
    return (pool[3] in (64, 128) and cache.key_pool.dtype in (torch.bfloat16, torch.float16)
            and pool[1] % 16 == 0 and pools_by_tma(cache))


def _bound(cache: PagedKVCache, max_context):
    if max_context is not None:
        return int(max_context)
    n = int(cache.seq_lengths.max()) if cache.seq_lengths.numel() else 0
    if n > cache.block_table.shape[1] * cache.block_size:
        raise ValueError(f"a sequence length ({n}) exceeds max_blocks_per_seq * block_size "
                         f"({cache.block_table.shape[1]} * {cache.block_size})")
    return n


def cast(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return x if x.dtype == dtype else x.to(dtype)


def _params(query, dims, cache: PagedKVCache, max_context: int):
    """(PagedParams, out, tensors that the call reads); ``dims`` as _check_query returns them."""
    n, hq, t, d, (nb, bs, hkv, _), (_, width) = dims
    kp = cache.key_pool
    q = cast(query, kp.dtype).contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    out = torch.empty_like(q)
    bt, sl = cache.block_table.contiguous(), cache.seq_lengths.contiguous()
    p = _lib.PagedParams(dtype_code(kp.dtype), n, hq, hkv, d, t, nb, bs, width, min(max_context, width * bs),
                         q.data_ptr(), kp.data_ptr(), cache.value_pool.data_ptr(), bt.data_ptr(),
                         sl.data_ptr(), out.data_ptr(), _scale(d))
    return p, out, (q, bt, sl)


@functools.lru_cache(maxsize=None)
def _scale(head_dim: int) -> float:
    return softmax_scale(head_dim)


def _workspace(p, nbytes: int, device):
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
        return ws
    return None


def paged_window_attention(query, cache: PagedKVCache, *, window_size: int, num_sinks: int = 0, max_context=None):
    """Sliding-window decode with sinks: ``query (B, Hq, T, D)`` -> same shape and type.

    Row ``t`` of sequence ``b`` stands at position ``seq_lengths[b] - T + t``
    (append the T tokens' K/V first) and sees the keys ``kv <= position`` with
    ``position - kv < window_size`` or ``kv < num_sinks``.  Rows in front of
    the sequence (T > its length) and empty sequences give zeros.  Pages that
    no row sees are not read: their table entries may be -1 (``free_window``).

    With ``max_context`` (an upper bound of the lengths) there is no host
    sync; a longer sequence is then cut to the planned splits and noted in
    ``_lib.device_status()``, as in ``paged_attention_batched``.
    """
    if window_size <= 0:
        raise ValueError(f"window_size must be positive, got {window_size}")
    if num_sinks < 0:
        raise ValueError(f"num_sinks must not be negative, got {num_sinks}")
    n, hq, t, d, pool, _ = dims = _check_query(query, cache)
    _need_cuda(query, cache)
    if n == 0 or t == 0:
        return torch.zeros_like(query)
    if not _fused(cache, pool):
        refuse_codes(cache)
        _bound(cache, None)
        return _window_by_sequence(query, cache, int(window_size), int(num_sinks))
    lib = _lib.load()
    p, out, keep = _params(query, dims, cache, _bound(cache, max_context))
    w, s = min(int(window_size), 1 << 40), min(int(num_sinks), 1 << 40)
    ws = _workspace(p, lib.attn_paged_window_workspace_size(C.byref(p), w, s), query.device)
    _lib.run("attn_paged_window", query.device, C.byref(p), w, s)
    del ws, keep
    return cast(out, query.dtype)


def _window_by_sequence(query, cache, window, sinks):
    out = torch.zeros_like(query)
    t = query.shape[2]
    for b in range(query.shape[0]):
        k, v, n = gather_window(cache, b, t, window, sinks)
        if n is None:
            continue
        kv = n  # positions of the gathered keys
        length = int(cache.seq_lengths[b])
        rows = torch.arange(length - t, length, device=query.device)
        dist = rows[:, None] - kv[None, :]
        mask = (dist >= 0) & ((dist < window) | (kv < sinks)[None, :])
        first = max(0, t - length)  # rows in front of the sequence keep their zeros
        out[b, :, first:] = attention(query[b:b + 1, :, first:].to(k.dtype), k, v, mask=mask[first:])[0].to(query.dtype)
    return out


def gather_window(cache: PagedKVCache, sequence_idx: int, rows: int, window: int, sinks: int):
    """Contiguous ``(1, Hkv, n, D)`` keys/values of the positions that the last ``rows`` rows see, and the positions."""
    length = int(cache.seq_lengths[sequence_idx])
    if length == 0:
        return None, None, None
    dev = cache.key_pool.device
    lo = max(0, length - rows - window + 1)
    pos = torch.cat([torch.arange(min(sinks, lo), device=dev), torch.arange(lo, length, device=dev)])
    k, v = (x.permute(1, 0, 2)[None].contiguous() for x in gather_positions(cache, sequence_idx, pos))
    return k, v, pos


def _tma_ready(x: torch.Tensor) -> torch.Tensor:
    """Unit stride on head_dim, other strides and the base in 16-byte steps (dimensions of one are not stepped)."""
    a, b, c, unit = x.stride()
    na, nb, nc, _ = x.shape
    ok = (unit == 1 and x.data_ptr() % 16 == 0 and (na == 1 or (a > 0 and a % 8 == 0))
          and (nb == 1 or (b > 0 and b % 8 == 0)) and (nc == 1 or (c > 0 and c % 8 == 0)))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def paged_tree_attention(query, draft_keys, draft_values, cache: PagedKVCache, parents, *, tree_lengths=None,
                         max_context=None):
    """Attention of drafted tokens: ``query (B, Hq, T, D)`` -> same shape and type.

    ``draft_keys``/``draft_values`` ``(B, Hkv, T, D)`` are the drafts' own K/V
    (any strides; not in the cache), ``parents (B, T)`` int32 gives each
    token's parent: an earlier token, or a negative number for a token that
    continues the context itself.  Row ``t`` sees the whole context
    (``seq_lengths[b]`` tokens), itself and its ancestors.  With
    ``tree_lengths (B,)`` the tokens at or past a sequence's length are
    padding: nothing sees them, their rows are zeros and their parents are not
    looked at.  A parent that is not
    in front of its token counts as negative and is noted in
    ``_lib.device_status()`` (``NOTICE_TREE_ORDER``).  T is at most 1024.

    ``max_context`` as in :func:`paged_window_attention`.  The accepted path
    goes into the cache with ``append_accepted``.
    """
    n, hq, t, d, pool, _ = dims = _check_query(query, cache)
    for name, x in (("draft_keys", draft_keys), ("draft_values", draft_values)):
        if not isinstance(x, torch.Tensor) or x.shape != (n, pool[2], t, d):
            raise ValueError(f"{name} must have shape {(n, pool[2], t, d)}, got "
                             f"{tuple(getattr(x, 'shape', ()))}")
        if x.device != query.device:
            raise RuntimeError(f"{name} must be on the query's device")
    dev = query.device
    parents = on_device(parents, dev)
    if parents.shape != (n, t):
        raise ValueError(f"parents must have shape {(n, t)}, got {tuple(parents.shape)}")
    if tree_lengths is not None:
        tree_lengths = on_device(tree_lengths, dev)
        if tree_lengths.shape != (n,):
            raise ValueError(f"tree_lengths must have shape {(n,)}, got {tuple(tree_lengths.shape)}")
    if t > 1024:
        raise NotImplementedError(f"{t} drafted tokens; at most 1024")
    _need_cuda(query, cache)
    if n == 0 or t == 0:
        return torch.zeros_like(query)
    if not _fused(cache, pool):
        refuse_codes(cache)
        _bound(cache, None)
        return _tree_by_sequence(query, draft_keys, draft_values, cache, parents, tree_lengths)
    lib = _lib.load()
    p, out, keep = _params(query, dims, cache, _bound(cache, max_context))
    dk, dv = (_tma_ready(cast(x, cache.key_pool.dtype)) for x in (draft_keys, draft_values))
    tr = _lib.PagedTree(dk.data_ptr(), dv.data_ptr(), dk.stride()[:3], dv.stride()[:3], parents.data_ptr(),
                        None if tree_lengths is None else tree_lengths.data_ptr())
    ws = _workspace(p, lib.attn_paged_tree_workspace_size(C.byref(p)), dev)
    _lib.run("attn_paged_tree", dev, C.byref(p), C.byref(tr))
    del ws, keep
    return cast(out, query.dtype)


def _tree_by_sequence(query, dk, dv, cache, parents, tree_lengths):
    out = torch.zeros_like(query)
    par = parents.tolist()
    lens = [query.shape[2]] * query.shape[0] if tree_lengths is None else tree_lengths.tolist()
    for b in range(query.shape[0]):
        m = min(max(lens[b], 0), query.shape[2])
        if m == 0:
            continue
        keys, values, n = gather_kv(cache, b)
        see = torch.zeros(m, n + m, dtype=torch.bool)
        see[:, :n] = True
        for t in range(m):
            if 0 <= par[b][t] < t:
                see[t, n:] = see[par[b][t], n:]
            see[t, n + t] = True
        k = torch.cat([keys.permute(1, 0, 2), dk[b, :, :m].to(keys.dtype)], 1)[None]
        v = torch.cat([values.permute(1, 0, 2), dv[b, :, :m].to(keys.dtype)], 1)[None]
        o = attention(query[b:b + 1, :, :m].to(k.dtype), k.contiguous(), v.contiguous(), mask=see.to(query.device))
        out[b, :, :m] = o[0].to(query.dtype)
    return out
