"""Paged caches in 8 bits, tokens into and out of paged caches, and attention over 8-bit pages.

``QuantizedPagedKVCache`` is :class:`PagedKVCache` with pools of ``torch.float8_e4m3fn`` or ``torch.int8`` and a
float32 scale for each page and kv head: a code stands for ``code * scale``.  Scales are powers of two, the least
one that brings the page's largest magnitude into the type (between 2^-100 and the largest for which code * scale
is finite; magnitudes beyond saturate), so each value is rounded once.

``append_tokens`` puts a whole padded batch of new tokens into either kind of cache, keys (and the queries beside
them) turned by their positions on the way; ``gather_tokens`` reads them back; ``paged_quantized_attention`` is the
decode over 8-bit pages.  No counterparts in the reference, which appends one sequence at a time and rotates in
passes of its own (attnax/paged_cache.py:144-198, attnax/attention.py:340-381).  Nothing here waits for the GPU
unless its docstring says so.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._spec import dtype_code
from .paged import PagedKVCache
from .paged_rows import _bound, _scale, check_tables, on_device, paged_window_attention
from .rotary import RotaryPlan, check_plan, plan_spec, rows_like, unit_stride

_FORMATS = {torch.float8_e4m3fn: _lib.POOL_E4M3, torch.int8: _lib.POOL_INT8}


@dataclass(frozen=True)
class QuantizedPagedKVCache:
    """Pools of 8-bit codes ``(num_blocks, block_size, num_kv_heads, head_dim)``, float32 scales
    ``(num_blocks, num_kv_heads)`` (not negative), block table and lengths as :class:`PagedKVCache` has them."""

    key_pool: torch.Tensor
    value_pool: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    block_table: torch.Tensor
    seq_lengths: torch.Tensor

    @property
    def num_blocks(self) -> int:
        return int(self.key_pool.shape[0])

    @property
    def block_size(self) -> int:
        return int(self.key_pool.shape[1])

    @property
    def num_kv_heads(self) -> int:
        return int(self.key_pool.shape[2])

    @property
    def head_dim(self) -> int:
        return int(self.key_pool.shape[3])


def init_quantized_paged_kv_cache(*, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                                  batch_size: int, max_blocks_per_seq: int, dtype=torch.float8_e4m3fn,
                                  device="cuda") -> QuantizedPagedKVCache:
    """Zero codes, scales of one, ``-1`` block table, zero lengths (as ``init_paged_kv_cache``)."""
    if dtype not in _FORMATS:
        raise ValueError(f"unsupported dtype {dtype}; expected float8_e4m3fn or int8")
    shape = (num_blocks, block_size, num_kv_heads, head_dim)
    kp, vp = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.ones(num_blocks, num_kv_heads, dtype=torch.float32, device=device) for _ in range(2))
    return QuantizedPagedKVCache(kp, vp, ks, vs,
                                 torch.full((batch_size, max_blocks_per_seq), -1, dtype=torch.int32, device=device),
                                 torch.zeros(batch_size, dtype=torch.int32, device=device))


def check_cache(cache):
    """(pool shape, table shape, pool format) of either kind of cache, its tensors checked."""
    if not isinstance(cache, (PagedKVCache, QuantizedPagedKVCache)):
        raise ValueError("cache must be a PagedKVCache or a QuantizedPagedKVCache")
    pool, rows = check_tables(cache)
    dev = cache.key_pool.device
    if isinstance(cache, QuantizedPagedKVCache):
        fmt = _FORMATS.get(cache.key_pool.dtype)
        if fmt is None:
            raise ValueError(f"unsupported pool dtype {cache.key_pool.dtype}; expected float8_e4m3fn or int8")
        want = (pool[0], pool[2])
        for name, x in (("key_scales", cache.key_scales), ("value_scales", cache.value_scales)):
            if x.shape != want or x.dtype != torch.float32:
                raise ValueError(f"{name} must be float32 {want}, got {x.dtype} {tuple(x.shape)}")
            if x.device != dev:
                raise RuntimeError(f"{name} must be on the pools' device")
            if not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    else:
        fmt = dtype_code(cache.key_pool.dtype)
    if not (cache.key_pool.is_contiguous() and cache.value_pool.is_contiguous()):
        raise ValueError("the pools must be contiguous")
    return pool, rows, fmt


def _need_cuda(cache):
    if not cache.key_pool.is_cuda:
        raise RuntimeError("attnax_b200 kernels need CUDA tensors; there is no CPU path")


def _scales(cache):
    if isinstance(cache, QuantizedPagedKVCache):
        return cache.key_scales.data_ptr(), cache.value_scales.data_ptr()
    return 0, 0


def with_table(cache, table: torch.Tensor, lengths: torch.Tensor):
    """The cache with another table and lengths: a QuantizedPagedKVCache, or a PagedKVCache of whatever has the fields
    of one (without the host time of dataclasses.replace and of a frozen constructor)."""
    if isinstance(cache, QuantizedPagedKVCache):
        new = object.__new__(type(cache))
        new.__dict__.update(cache.__dict__, block_table=table, seq_lengths=lengths)
    else:
        new = object.__new__(PagedKVCache)
        new.__dict__.update(key_pool=cache.key_pool, value_pool=cache.value_pool, block_table=table,
                            seq_lengths=lengths)
    return new


_append_params = _lib.packer(_lib.PagedAppendParams)
_gather_params = _lib.packer(_lib.PagedGatherParams)
_attend_params = _lib.packer(_lib.PagedAttend8Params)
_NO_QUERY = (0, 0, 0, 0, 0, 0, 0, 0, 0)


def _check_append(cache, n: int, hk: int, d: int, keys, values, query, rotary):
    dev = cache.key_pool.device
    for name, x in (("keys", keys), ("values", values)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4 or x.shape[0] != n or x.shape[1] != hk or x.shape[3] != d:
            raise ValueError(f"{name} must have shape ({n}, {hk}, T, {d}), got {tuple(getattr(x, 'shape', ()))}")
        if x.device != dev:
            raise RuntimeError(f"{name} must be on the cache's device")
    if keys.shape != values.shape:
        raise ValueError(f"keys shape {tuple(keys.shape)} != values shape {tuple(values.shape)}")
    if keys.dtype != values.dtype:
        raise ValueError(f"keys are {keys.dtype}, values {values.dtype}")
    dtype_code(keys.dtype)
    t = keys.shape[2]
    if query is not None:
        if not isinstance(query, torch.Tensor) or query.dim() != 4 or query.shape[0] != n or query.shape[2] != t \
                or query.shape[3] != d:
            raise ValueError(f"query must have shape ({n}, Hq, {t}, {d}), got {tuple(getattr(query, 'shape', ()))}")
        if query.dtype != keys.dtype:
            raise ValueError(f"query is {query.dtype}, keys {keys.dtype}")
        if query.device != dev:
            raise RuntimeError("query must be on the cache's device")
        if rotary is None:
            raise ValueError("query needs a rotary plan")
    if rotary is not None:
        check_plan(rotary, d, dev)
    _need_cuda(cache)


def append_tokens(cache, keys: torch.Tensor, values: torch.Tensor, *, new_lengths=None,
                  rotary: RotaryPlan | None = None, query: torch.Tensor | None = None, check: bool = True):
    """Appends a padded batch of new tokens to their sequences' pages, in one launch.

    ``keys``/``values (B, Hkv, T, D)`` (any strides; bf16, fp16 or fp32) hold T tokens per sequence, of which the
    first ``new_lengths[b]`` count (default: all).  Token ``i`` goes to position ``seq_lengths[b] + i``, whose page
    ``allocate_blocks`` has put into the table.  With ``rotary`` the keys are turned by that position, and so is
    ``query (B, Hq, T, D)`` if given (row ``i``, padding rows too).  ``cache`` is a :class:`PagedKVCache` or a
    :class:`QuantizedPagedKVCache`; pools and scales are written in place.  Returns the cache with its new lengths,
    with a query ``(cache, query')``.

    An 8-bit page that gets tokens keeps the larger of its scale and the one that they need, and its older codes
    are restated where it grows (e4m3 codes keep their values unless they become subnormal, int8 codes round once
    more).  Infinities and NaN are stored as NaN; in an int8 page, which has none, the whole page reads as NaN
    until it is begun anew.  A page that gets tokens must belong to one sequence (``fork_sequences`` shares full
    pages only).  What is written and returned carries no gradient.

    ``check=True`` waits for the GPU and raises ``ValueError`` before anything is written if a length or a page is
    missing or out of range; with ``check=False`` there is no wait, and such tokens (all of a sequence whose length is
    negative) are skipped and noted in ``_lib.device_status()`` (``NOTICE_PAGE_LIST``; lengths still count them).
    """
    pool, (n, width), fmt = check_cache(cache)
    kp, vp = cache.key_pool, cache.value_pool
    dev = kp.device
    _check_append(cache, n, pool[2], pool[3], keys, values, query, rotary)
    if new_lengths is not None:
        new_lengths = on_device(new_lengths, dev)
        if new_lengths.shape != (n,):
            raise ValueError(f"new_lengths must have shape ({n},), got {tuple(new_lengths.shape)}")
    t = keys.shape[2]
    if n == 0 or t == 0:
        if check and n and new_lengths is not None and bool((new_lengths != 0).any()):
            raise ValueError("new_lengths counts tokens that are not there")
        return cache if query is None else (cache, torch.empty_like(query))
    k, v = unit_stride(keys), unit_stride(values)
    bt, sl = cache.block_table.contiguous(), cache.seq_lengths.contiguous()
    q_out, q_args = None, _NO_QUERY
    if query is not None:
        q = unit_stride(query)
        q_out = rows_like(q)
        q_args = (q.shape[1], q.data_ptr(), q_out.data_ptr(), *q.stride()[:3], *q_out.stride()[:3])
    p = _append_params(dtype_code(keys.dtype), fmt, *pool, kp.data_ptr(), vp.data_ptr(), *_scales(cache), n, width,
                       bt.data_ptr(), sl.data_ptr(), k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], t,
                       0 if new_lengths is None else new_lengths.data_ptr(), *plan_spec(rotary), *q_args, 0, 0)
    if check:
        bad = torch.full((), 2**31 - 1, dtype=torch.int32, device=dev)
        p.bad = bad.data_ptr()
        _lib.run("attn_paged_append_tokens", dev, C.byref(p))
        if int(bad) != 2**31 - 1:
            raise ValueError(f"sequence {int(bad)}: its count of new tokens or the page for one is out of range; call "
                             "allocate_blocks before append_tokens")
        p.bad = None
    out = torch.empty_like(sl)
    p.lengths_out = out.data_ptr()
    _lib.run("attn_paged_append_tokens", dev, C.byref(p))
    del bt, sl, k, v
    new = with_table(cache, cache.block_table, out)
    return new if query is None else (new, q_out)


def _gather(cache, pool, rows, fmt, starts, count: int, dtype):
    n, width = rows
    dev = cache.key_pool.device
    bt, sl = cache.block_table.contiguous(), cache.seq_lengths.contiguous()
    k = torch.empty((n, count, pool[2], pool[3]), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    p = _gather_params(dtype_code(dtype), fmt, *pool, cache.key_pool.data_ptr(), cache.value_pool.data_ptr(),
                       *_scales(cache), n, width, bt.data_ptr(), sl.data_ptr(),
                       0 if starts is None else starts.data_ptr(), count, k.data_ptr(), v.data_ptr())
    _lib.run("attn_paged_gather_tokens", dev, C.byref(p))
    del bt, sl
    return k, v


def gather_tokens(cache, starts, count: int, *, dtype=None):
    """``(keys, values)``, each ``(B, Hkv, count, D)``: positions ``starts[b] .. starts[b] + count - 1`` of every
    sequence, the batched form of ``gather_kv`` for both kinds of cache.

    ``starts (B,)`` integers, or ``None`` for the beginning; positions outside a sequence give zeros, and so do those
    whose page is missing (``free_window``), noted in ``_lib.device_status()`` (``NOTICE_PAGE_LIST``).  8-bit codes
    come back as the values that they stand for, rounded to ``dtype`` (default: the pools' type; bfloat16 for 8-bit
    pools, which holds every code times a power of two exactly).  Nothing waits for the GPU.
    """
    pool, rows, fmt = check_cache(cache)
    if dtype is None:
        dtype = torch.bfloat16 if isinstance(cache, QuantizedPagedKVCache) else cache.key_pool.dtype
    dtype_code(dtype)
    count = int(count)
    if count < 0:
        raise ValueError(f"count must not be negative, got {count}")
    dev = cache.key_pool.device
    if starts is not None:
        starts = on_device(starts, dev)
        if starts.shape != (rows[0],):
            raise ValueError(f"starts must have shape ({rows[0]},), got {tuple(starts.shape)}")
    _need_cuda(cache)
    k, v = _gather(cache, pool, rows, fmt, starts, count, dtype)
    return k.transpose(1, 2), v.transpose(1, 2)


def paged_quantized_attention(query: torch.Tensor, cache: QuantizedPagedKVCache, *, max_context=None) -> torch.Tensor:
    """Attention of the last positions over 8-bit pages: ``query (B, Hq, T, D)`` -> same shape and type.

    Row ``t`` of sequence ``b`` stands at position ``seq_lengths[b] - T + t`` (append the T tokens first) and sees
    the keys up to it.  Rows in front of the sequence (T > its length) and empty sequences give zeros.  bf16, fp16
    or fp32 queries; products in fp16 on codes that fp16 holds exactly, with scales and softmax in fp32.  The query
    is scaled by a power of two per row and held in fp16: exact for 16-bit types down to 2^-28 of the row's largest
    channel, and off by at most 2^-39 of that below; the channels of an fp32 query are rounded to 11 bits.  So are
    the weights that meet the values.  An fp32 result is therefore good to about 11 bits (other caches, below: all).

    Rows that stand behind a page which is missing (taken by ``free_window``, or out of range) are NaN, noted in
    ``_lib.device_status()`` (``NOTICE_PAGE_LIST``): there is no window here that would leave such pages out.

    With ``max_context`` (an upper bound of the lengths) there is no host sync; a longer sequence is then cut to
    the planned splits and noted in ``_lib.device_status()``, as in ``paged_attention_batched``.  head_dim 64 or
    128, a block size that is a multiple of 16 and pools that start on 16 bytes take the fused kernel; other caches
    are brought to bf16 or fp32 (``gather_tokens``), then attended as ``paged_window_attention`` does, waiting for the
    lengths (``NotImplementedError`` for head dims that the flash kernels do not have).  For inference: what it
    returns carries no gradient.
    """
    if not isinstance(cache, QuantizedPagedKVCache):
        raise ValueError("cache must be a QuantizedPagedKVCache (paged_attention_batched takes the other one)")
    if not isinstance(query, torch.Tensor) or query.dim() != 4:
        raise ValueError("query must be (num_seqs, num_heads, seq_q, head_dim)")
    n, hq, t, d = query.shape
    pool, rows, fmt = check_cache(cache)
    if n != rows[0]:
        raise ValueError(f"query has {n} sequences, the cache {rows[0]}")
    if hq % pool[2] != 0:
        raise ValueError(f"num_heads ({hq}) must be divisible by num_kv_heads ({pool[2]})")
    if d != pool[3]:
        raise ValueError(f"query head_dim {d} != cache head_dim {pool[3]}")
    code = dtype_code(query.dtype)
    dev = cache.key_pool.device
    if not query.is_cuda or query.device != dev:
        raise RuntimeError("attnax_b200 kernels need the query on the cache's CUDA device; there is no CPU path")
    if n == 0 or t == 0 or hq == 0:
        return torch.zeros_like(query)
    nb, bs, hk, _ = pool
    kp, vp = cache.key_pool, cache.value_pool
    if d not in (64, 128) or bs % 16 or (kp.data_ptr() | vp.data_ptr()) % 16:
        return _attend_gathered(query, cache, pool, rows, fmt)
    q = query.contiguous()
    if q.data_ptr() % 16:  # (vector loads)
        q = q.clone()
    out = torch.empty_like(q)
    bt, sl = cache.block_table.contiguous(), cache.seq_lengths.contiguous()
    ctx = min(max(_bound(cache, max_context), 0), rows[1] * bs, 2**31 - 1)
    p = _attend_params(code, fmt, n, hq, hk, d, t, nb, bs, rows[1], ctx, q.data_ptr(), kp.data_ptr(), vp.data_ptr(),
                       cache.key_scales.data_ptr(), cache.value_scales.data_ptr(), bt.data_ptr(), sl.data_ptr(),
                       out.data_ptr(), _scale(d), 0, 0)
    nbytes = _lib.load().attn_paged_attend8_workspace_size(C.byref(p))
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    _lib.run("attn_paged_attend8", dev, C.byref(p))
    return out


def _attend_gathered(query, cache, pool, rows, fmt):
    """The sequences in bf16 (exact for scales that are powers of two) or fp32, one behind the other, each on pages of its own, and the window kernels."""
    longest = max(_bound(cache, None), 1)
    n, t = rows[0], query.shape[2]
    _, _, hk, d = pool
    dtype = torch.bfloat16 if query.dtype == torch.bfloat16 else torch.float32  # (fp16 does not hold every scale)
    size = -(-longest // 16) * 16
    k, v = _gather(cache, pool, rows, fmt, None, size, dtype)
    pos = torch.arange(size, dtype=torch.int32, device=query.device)
    entry = cache.block_table[:, (pos // pool[1]).clamp(max=rows[1] - 1).long()]
    missing = ((entry < 0) | (entry >= pool[0])) & (pos < cache.seq_lengths[:, None])
    k[..., 0].masked_fill_(missing[:, :, None], float("nan"))  # (such tokens came back as zeros)
    table = torch.arange(n * (size // 16), dtype=torch.int32, device=query.device).view(n, size // 16)
    wide = PagedKVCache(k.view(-1, 16, hk, d), v.view(-1, 16, hk, d), table, cache.seq_lengths)
    return paged_window_attention(query, wide, window_size=size + t, max_context=longest)
