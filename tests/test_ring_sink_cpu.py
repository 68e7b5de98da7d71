"""Ring schedule with a sink window on CPU ranks (gloo): forward and gradients of the global sequence.

The schedule sees the chain as causal (a sink is kept at any distance), so no
hop that holds sinks is dropped; the window and the sinks themselves go by
global positions inside each chunk pair.
"""

import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import attnax_b200 as ax
import oracle as O
from attnax_b200._spec import band_of
from tests.test_ring_cpu import OracleOps, _free_port

WINDOW, SINKS = 7, 3


def sink_window(scores, b_idx, h_idx, q_idx, kv_idx):
    keep = (kv_idx <= q_idx) & ((q_idx - kv_idx < WINDOW) | (kv_idx < SINKS))
    return np.where(keep, scores, np.finfo(scores.dtype).min)


def _worker(rank, world, port, q, k, v, do, out, grads):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from attnax_b200._ring_impl import RingSchedule, ring_schedule_backward, ring_schedule_forward

        S = q.shape[2] // world
        sl = slice(rank * S, (rank + 1) * S)
        band = band_of(ax.sink_window_mod(WINDOW, SINKS))
        for zigzag in (False, True):
            sched = RingSchedule(world, rank, S, zigzag)
            ops = OracleOps(None, sink_window, None, q.shape[1], k.shape[1])
            tq, tk, tv, tdo = (torch.from_numpy(np.ascontiguousarray(x[:, :, sl])).double() for x in (q, k, v, do))
            st = {}
            got, _ = ring_schedule_forward(tq, tk, tv, ops=ops, sched=sched, band=band, state=st)
            np.testing.assert_allclose(got.numpy(), out[:, :, sl], atol=1e-10, rtol=1e-10)
            res = ring_schedule_backward(st["q"], st["k"], st["v"], st["out"], st["lse"], tdo, ops=ops, sched=sched,
                                         band=band)
            for g, w in zip(res, grads):
                # (1e-6: the oracle's closed-form backward rounds the scale to float32)
                np.testing.assert_allclose(g.numpy(), w[:, :, sl], atol=1e-6, rtol=1e-6)
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_ring_schedule_with_sinks(world):
    rng = np.random.default_rng(world)
    B, Hq, Hkv, S, D = 1, 4, 2, 16 * world, 8
    q, k, v, do = (rng.standard_normal((B, h, S, D)) for h in (Hq, Hkv, Hkv, Hq))
    out = O.gqa_attention(q, k, v, score_mod=sink_window)
    grads = O.gqa_attention_bwd(q, k, v, do, score_mod=sink_window)
    mp.spawn(_worker, args=(world, _free_port(), q, k, v, do, out, grads), nprocs=world, join=True)


def test_the_library_ring_does_not_take_sinks():
    """attn_ring_fwd knows bands only: a sink window runs the host schedule."""
    from attnax_b200 import _ring_capi

    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16)
    assert _ring_capi.eligible(q, q, q, ax.sliding_window_mod(4), None)
    assert not _ring_capi.eligible(q, q, q, ax.sink_window_mod(4, 2), None)
