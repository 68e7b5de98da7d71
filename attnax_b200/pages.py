"""Operators on the pages of a :class:`PagedKVCache`: accept, copy, fork, free and compact.

They take whole batches and return new ``PagedKVCache`` objects like the rest
of the paged API (``allocate_blocks``, ``append_kv``); tables and lengths are
new tensors, the pools are written in place and shared.  Nothing here waits
for the GPU unless it says so: counts come back as 0-d int32 tensors on the
cache's device, lists of pages as int32 tensors padded with -1, ready for
``allocate_blocks(free_block_ids=...)``.

Index arguments may be Python sequences or CPU tensors, which are checked on
the host (``ValueError``), or int32 tensors on the device, where an entry that
cannot be used is skipped and noted in ``_lib.device_status()``
(``NOTICE_PAGE_LIST``).  No counterparts in the reference, which allocates and
appends one sequence at a time (attnax/paged_cache.py:92-198).
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._spec import dtype_code
from .paged import PagedKVCache
from .paged_rows import cast, check_tables, narrow, on_device


_Strides = C.c_int64 * 3


def _params(cache: PagedKVCache):
    """(PagedCacheParams, tensors it points into)."""
    pool, rows = check_tables(cache)
    kp, vpool = cache.key_pool, cache.value_pool
    if not kp.is_cuda:
        raise RuntimeError("attnax_b200 kernels need CUDA tensors; there is no CPU path")
    if not (kp.is_contiguous() and vpool.is_contiguous()):
        raise ValueError("page operators write the pools in place and need them contiguous")
    bt, sl = cache.block_table.contiguous(), cache.seq_lengths.contiguous()
    p = _lib.PagedCacheParams(dtype_code(kp.dtype), *pool, kp.data_ptr(), vpool.data_ptr(), *rows,
                              bt.data_ptr(), sl.data_ptr())
    return p, (bt, sl)


def _indices(x, device, limit: int, what: str, distinct: bool = False) -> torch.Tensor:
    """int32 indices on the device; what comes from the host is checked there."""
    t = x if isinstance(x, torch.Tensor) else torch.as_tensor(x)
    if t.dim() != 1:
        raise ValueError(f"{what} must be one-dimensional, got shape {tuple(t.shape)}")
    if t.is_cuda and t.dtype == torch.int32 and t.device == device:
        return t.contiguous()
    if t.numel() and (t.is_floating_point() or t.dtype == torch.bool):
        raise ValueError(f"{what} must be integers, got {t.dtype}")
    if not t.is_cuda:
        bad = (t < 0) | (t >= limit)
        if bool(bad.any()):
            raise ValueError(f"{what} has entry {int(t[bad][0])}, outside [0, {limit})")
        if distinct and t.unique().numel() != t.numel():
            raise ValueError(f"{what} names an index twice")
    return narrow(t, device)


def copy_blocks(cache: PagedKVCache, src_blocks, dst_blocks) -> PagedKVCache:
    """Copies page ``src_blocks[i]`` over page ``dst_blocks[i]`` (keys and values), in place.

    The entries run in no order: a destination must be named once and must not
    be a source of another entry (``ValueError`` for host lists; on the device
    such an entry is skipped and noted, the first of equal destinations wins).
    """
    dev, nb = cache.key_pool.device, cache.num_blocks
    src = _indices(src_blocks, dev, nb, "src_blocks")
    dst = _indices(dst_blocks, dev, nb, "dst_blocks", distinct=True)
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source pages for {dst.numel()} destinations")
    if not any(isinstance(x, torch.Tensor) and x.is_cuda for x in (src_blocks, dst_blocks)):
        s, d = torch.as_tensor(src_blocks), torch.as_tensor(dst_blocks)
        both = d[s != d][torch.isin(d[s != d], s)]
        if both.numel():
            raise ValueError(f"page {int(both[0])} is both a source and a destination")
    p, keep = _params(cache)
    if src.numel():
        _lib.run("attn_paged_copy", dev, C.byref(p), src.data_ptr(), dst.data_ptr(), src.numel())
    del keep
    return cache


def fork_sequences(cache: PagedKVCache, src_sequences, dst_sequences, free_block_ids):
    """Rows ``dst_sequences[i]`` become copies of rows ``src_sequences[i]``: ``(cache, used)``.

    Full pages are shared; a last page that is not full is copied to the next
    of ``free_block_ids``, so source and copy can both append.  ``used`` (0-d
    int32 on the device) is the number of ids taken from the front of the
    list.  Pages that only a replaced row held are not freed (call
    ``free_sequences`` first).  With fewer ids than forks this waits for the
    lengths and raises ``ValueError`` if they are too few.

    On the device: ids that are no pages, or are listed again, leave the copy
    with its full pages and a note; of forks onto one row the first wins, the
    others are skipped and noted.  ``used`` counts the ids of such forks too
    (compare the new table with the list to have those pages back).
    """
    dev = cache.key_pool.device
    n_seq = cache.block_table.shape[0]
    src = _indices(src_sequences, dev, n_seq, "src_sequences")
    dst = _indices(dst_sequences, dev, n_seq, "dst_sequences", distinct=True)
    free = _indices(free_block_ids, dev, cache.num_blocks, "free_block_ids", distinct=True)
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source rows for {dst.numel()} destinations")
    if src.numel() == 0:
        return cache, torch.zeros((), dtype=torch.int32, device=dev)
    if free.numel() < src.numel():
        ok = (src >= 0) & (src < n_seq)
        need = int((cache.seq_lengths[src[ok].long()] % cache.block_size != 0).sum())
        if need > free.numel():
            raise ValueError(f"free_block_ids has {free.numel()} entries but {need} are needed")
    p, keep = _params(cache)
    table = torch.empty(cache.block_table.shape, dtype=torch.int32, device=dev)
    lens = torch.empty(cache.seq_lengths.shape, dtype=torch.int32, device=dev)
    used = torch.empty((), dtype=torch.int32, device=dev)
    _lib.run("attn_paged_fork", dev, C.byref(p), src.data_ptr(), dst.data_ptr(), src.numel(),
          free.data_ptr() if free.numel() else None, free.numel(), table.data_ptr(), lens.data_ptr(), used.data_ptr())
    del keep
    return PagedKVCache(cache.key_pool, cache.value_pool, table, lens), used


def _scratch(ws):
    return (None, 0) if ws is None else (ws.data_ptr(), ws.numel())


def _freed(cache: PagedKVCache, p):
    dev = cache.key_pool.device
    nbytes = _lib.load().attn_paged_free_workspace_size(C.byref(p))  # 0 but for huge pools
    return (torch.empty(cache.block_table.shape, dtype=torch.int32, device=dev),
            torch.empty(cache.num_blocks, dtype=torch.int32, device=dev),
            torch.empty((), dtype=torch.int32, device=dev),
            torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None)


def free_sequences(cache: PagedKVCache, sequences):
    """Ends rows: ``(cache, freed_block_ids, num_freed)``.

    The rows get -1 entries and length 0.  ``freed_block_ids``
    ``(num_blocks,)`` lists the pages that only these rows referred to, in
    ascending order, padded with -1; pages that other rows share stay.
    """
    dev = cache.key_pool.device
    seqs = _indices(sequences, dev, cache.block_table.shape[0], "sequences")
    p, keep = _params(cache)
    table, freed, count, ws = _freed(cache, p)
    lens = torch.empty(cache.seq_lengths.shape, dtype=torch.int32, device=dev)
    _lib.run("attn_paged_free", dev, C.byref(p), seqs.data_ptr() if seqs.numel() else None, seqs.numel(),
          table.data_ptr(), lens.data_ptr(), freed.data_ptr(), count.data_ptr(), *_scratch(ws))
    del keep
    return PagedKVCache(cache.key_pool, cache.value_pool, table, lens), freed, count


def free_window(cache: PagedKVCache, *, window_size: int, num_sinks: int = 0):
    """Frees what ``paged_window_attention`` no longer reads: ``(cache, freed_block_ids, num_freed)``.

    A page goes when all its tokens lie behind the first ``num_sinks`` and in
    front of the window of the next token (position ``seq_lengths``); its entry
    becomes -1 and the lengths stay.  Whatever reads the whole context
    (``paged_attention``, ``paged_tree_attention``, ``gather_kv``) must not be
    used on such rows.
    """
    if window_size <= 0:
        raise ValueError(f"window_size must be positive, got {window_size}")
    if num_sinks < 0:
        raise ValueError(f"num_sinks must not be negative, got {num_sinks}")
    dev = cache.key_pool.device
    p, keep = _params(cache)
    table, freed, count, ws = _freed(cache, p)
    _lib.run("attn_paged_free_window", dev, C.byref(p), min(int(window_size), 1 << 40), min(int(num_sinks), 1 << 40),
          table.data_ptr(), freed.data_ptr(), count.data_ptr(), *_scratch(ws))
    del keep
    return PagedKVCache(cache.key_pool, cache.value_pool, table, cache.seq_lengths), freed, count


def compact_blocks(cache: PagedKVCache):
    """Moves the pages that rows refer to to the front of the pool: ``(cache, num_live)``.

    The pool is rewritten in place, so caches made before this call no longer
    describe it; pages ``[num_live, num_blocks)`` are free afterwards.  Live
    pages below ``num_live`` stay where they are; the others go, ascending, to
    the free pages below it, ascending.  Shared pages stay shared.
    """
    dev = cache.key_pool.device
    p, keep = _params(cache)
    table = torch.empty(cache.block_table.shape, dtype=torch.int32, device=dev)
    live = torch.empty((), dtype=torch.int32, device=dev)
    ws = torch.empty(_lib.load().attn_paged_compact_workspace_size(C.byref(p)), dtype=torch.uint8, device=dev)
    _lib.run("attn_paged_compact", dev, C.byref(p), table.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel())
    del keep
    return PagedKVCache(cache.key_pool, cache.value_pool, table, cache.seq_lengths), live


def append_accepted(cache: PagedKVCache, draft_keys, draft_values, accepted, accepted_lengths, *,
                    check: bool = True) -> PagedKVCache:
    """Appends each sequence's accepted drafts to its pages.

    ``draft_keys``/``draft_values`` ``(B, Hkv, T, D)`` are those of
    ``paged_tree_attention``; ``accepted (B, A)`` int32 holds draft indices in
    order of their positions, ``accepted_lengths (B,)`` how many of them count.
    Token ``accepted[b, i]`` goes to position ``seq_lengths[b] + i``, whose
    page ``allocate_blocks`` has put into the table.

    ``check=True`` waits for the GPU and raises ``ValueError`` before anything
    is written if an index, a length or a page is missing or out of range;
    with ``check=False`` there is no wait, and such tokens are skipped and
    noted (lengths still count them).
    """
    dev = cache.key_pool.device
    n = cache.block_table.shape[0]
    for name, x in (("draft_keys", draft_keys), ("draft_values", draft_values)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4 or x.shape[:2] != (n, cache.num_kv_heads) \
                or x.shape[3] != cache.head_dim:
            raise ValueError(f"{name} must have shape ({n}, {cache.num_kv_heads}, T, {cache.head_dim}), got "
                             f"{tuple(getattr(x, 'shape', ()))}")
        if x.device != dev:
            raise RuntimeError(f"{name} must be on the cache's device")
    if draft_keys.shape != draft_values.shape:
        raise ValueError(f"draft_keys shape {tuple(draft_keys.shape)} != draft_values shape "
                         f"{tuple(draft_values.shape)}")
    acc, lens = on_device(accepted, dev), on_device(accepted_lengths, dev)
    if acc.dim() != 2 or acc.shape[0] != n:
        raise ValueError(f"accepted must have shape ({n}, A), got {tuple(acc.shape)}")
    if lens.shape != (n,):
        raise ValueError(f"accepted_lengths must have shape ({n},), got {tuple(lens.shape)}")
    t = draft_keys.shape[2]
    p, keep = _params(cache)
    if n == 0 or t == 0 or acc.shape[1] == 0:
        if check and n and bool((lens != 0).any()):
            raise ValueError("accepted_lengths counts tokens that are not there")
        return cache
    kd, vd = cast(draft_keys, cache.key_pool.dtype), cast(draft_values, cache.key_pool.dtype)
    kd, vd = (x if x.stride(3) == 1 else x.contiguous() for x in (kd, vd))
    ks, vs = _Strides(*kd.stride()[:3]), _Strides(*vd.stride()[:3])
    args = (C.byref(p), kd.data_ptr(), vd.data_ptr(), ks, vs, t, acc.data_ptr(), acc.shape[1], lens.data_ptr())
    if check:
        bad = torch.full((), 2**31 - 1, dtype=torch.int32, device=dev)
        _lib.run("attn_paged_accept", dev, *args, None, bad.data_ptr())
        if int(bad) != 2**31 - 1:
            raise ValueError(f"sequence {int(bad)}: an accepted index, its count or the page for it is out of "
                             "range; call allocate_blocks before append_accepted")
    out = torch.empty(cache.seq_lengths.shape, dtype=torch.int32, device=dev)
    _lib.run("attn_paged_accept", dev, *args, out.data_ptr(), None)
    del keep
    return PagedKVCache(cache.key_pool, cache.value_pool, cache.block_table, out)
