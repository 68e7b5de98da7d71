"""Rotary positions with their gradient: both pair layouts, a part of the head, scaled frequencies.

``apply_rope`` / ``apply_rope_table`` are the reference's rotation (attnax/embeddings.py:126-184): split
halves of the whole head, cos/sin tables in the tensor's dtype, no gradient.  ``rotary_plan`` +
``apply_rotary`` have no counterpart there: frequencies are kept as 64-bit fixed-point fractions of a
turn, the kernel forms each angle from the position itself (exact for positions of any size, nothing is
read but the tensors), and queries and keys turn in one launch, forward and backward.
"""

from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._spec import differentiated, dtype_code


@dataclass(frozen=True)
class RotaryPlan:
    """What :func:`apply_rotary` and ``append_tokens`` turn by: made once by :func:`rotary_plan`, kept by the model."""

    turns: torch.Tensor  # int64 (rotary_dim // 2,): frequency / 2 pi as a fraction of 2^64 (the bits of a uint64)
    interleaved: bool
    magnitude: float

    @property
    def rotary_dim(self) -> int:
        return 2 * int(self.turns.shape[0])


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       low_factor: float = 1.0, high_factor: float = 4.0):
    """``(frequencies, magnitude)``: radians per position of each pair, float64 on the host, and the factor on both
    rotated tensors.

    ``w_i = base ** (-2 i / rotary_dim)``; ``scaling`` stretches them for contexts ``factor`` times as long:

    * ``"linear"``: ``w / factor`` (positions interpolated);
    * ``"ntk"``: the base becomes ``base * factor ** (rotary_dim / (rotary_dim - 2))``;
    * ``"yarn"``: pairs that turn more than ``beta_fast`` times within ``original_length`` keep their frequency,
      those below ``beta_slow`` turns get ``w / factor``, a linear ramp over the pair index between them (its ends
      rounded outwards and kept within ``0 .. rotary_dim - 1``);
      magnitude ``0.1 ln(factor) + 1`` (1 for factors up to 1);
    * ``"wavelength"``: by ``original_length`` over the wavelength: at or above ``high_factor`` the frequency stays,
      at or below ``low_factor`` it is ``w / factor``, linear in that quotient between them.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"base must be positive, got {base}")
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"factor must be positive, got {factor}")
    n = rotary_dim // 2
    i = torch.arange(n, dtype=torch.float64)
    w = float(base) ** (-i / n)
    if scaling is None:
        if factor != 1.0:
            raise ValueError("factor needs a scaling")
        return w, 1.0
    if scaling == "linear":
        return w / factor, 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("'ntk' needs a rotary_dim above 2")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-i / n), 1.0
    if scaling not in ("yarn", "wavelength"):
        raise ValueError(f"scaling must be 'linear', 'ntk', 'yarn' or 'wavelength', got {scaling!r}")
    if original_length is None or original_length <= 0:
        raise ValueError(f"{scaling!r} needs the original_length that the frequencies were trained for")
    if scaling == "yarn":
        if base <= 1.0 or not beta_fast > beta_slow > 0:
            raise ValueError("'yarn' needs a base above 1 and beta_fast > beta_slow > 0")

        def pair_of(turns):  # the (real) index of the pair that turns that often within original_length
            return rotary_dim * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1) if pair_of(beta_slow) > 0 else torch.ones_like(i)
        return w * (1 - ramp) + w / factor * ramp, 0.1 * math.log(max(factor, 1.0)) + 1.0
    if not high_factor > low_factor:
        raise ValueError("'wavelength' needs high_factor > low_factor")
    keep = ((original_length * w / (2 * math.pi) - low_factor) / (high_factor - low_factor)).clamp(0, 1)
    return w * keep + w / factor * (1 - keep), 1.0


def rotary_plan(rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False, scaling: str | None = None,
                device="cuda", **kw) -> RotaryPlan:
    """A plan for the first ``rotary_dim`` channels of each head; channels behind them are left as they are.

    ``interleaved=False`` pairs channel ``i`` with ``i + rotary_dim // 2``, ``True`` channel ``2 i`` with ``2 i + 1``.
    ``scaling`` and the other arguments are those of :func:`rotary_frequencies`.
    """
    w, magnitude = rotary_frequencies(rotary_dim, base=base, scaling=scaling, **kw)
    return rotary_plan_from_frequencies(w, interleaved=interleaved, magnitude=magnitude, device=device)


def rotary_plan_from_frequencies(frequencies, *, interleaved: bool = False, magnitude: float = 1.0,
                                 device="cuda") -> RotaryPlan:
    """A plan for given frequencies (radians per position, one per pair; read in 64 bits on the host)."""
    w = frequencies if isinstance(frequencies, torch.Tensor) else torch.as_tensor(frequencies, dtype=torch.float64)
    w = w.detach().to("cpu", torch.float64)
    if w.dim() != 1 or w.numel() == 0 or not bool(torch.isfinite(w).all()):
        raise ValueError("frequencies must be a non-empty list of finite numbers")
    bits = []
    for x in (w / (2 * math.pi)).tolist():  # whole turns per position fall away: positions are integers
        u = int(math.ldexp(x % 1.0, 64)) % 2**64
        bits.append(u - 2**64 if u >= 2**63 else u)
    return RotaryPlan(torch.tensor(bits, dtype=torch.int64, device=device), bool(interleaved), float(magnitude))


def check_plan(plan: RotaryPlan, head_dim: int, device):
    if not isinstance(plan, RotaryPlan):
        raise ValueError("plan must be a RotaryPlan (rotary_plan)")
    if plan.rotary_dim > head_dim:
        raise ValueError(f"the plan turns {plan.rotary_dim} channels, head_dim is {head_dim}")
    if plan.turns.dtype != torch.int64 or not plan.turns.is_contiguous():
        raise ValueError("the plan's turns must be contiguous int64")
    if plan.turns.device != device:
        raise RuntimeError(f"the plan is on {plan.turns.device}, the tensors on {device}")


def plan_spec(plan: RotaryPlan | None):
    """The flattened ``attn_rotary_spec_t``."""
    if plan is None:
        return 0, 0, 0, 1.0
    return plan.turns.data_ptr(), 2 * plan.turns.shape[0], plan.interleaved, plan.magnitude


def unit_stride(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def rows_like(x: torch.Tensor) -> torch.Tensor:
    """An output for ``x``, in its layout where that is dense.  (Views whose rows overlap have no such layout:
    ``empty_like`` may then put other axes inside the channels, which the kernels take for neighbours.)"""
    out = torch.empty_like(x)
    return out if out.stride(3) == 1 or x.shape[3] == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


_params = _lib.packer(_lib.RotaryParams)
_NO_STRIDES = (0, 0, 0)


def _launch(q, k, turns, interleaved, magnitude, positions, inverse):
    """Turned copies of ``q`` and ``k`` (or ``None``), laid out like them."""
    q = unit_stride(q)
    q_out = rows_like(q)
    b, hq, s, d = q.shape
    if k is None:
        k_out, hk, kp, kop, ks, kos = None, 0, 0, 0, _NO_STRIDES, _NO_STRIDES
    else:
        k = unit_stride(k)
        k_out = rows_like(k)
        hk, kp, kop, ks, kos = k.shape[1], k.data_ptr(), k_out.data_ptr(), k.stride()[:3], k_out.stride()[:3]
    if positions is None:
        pos, wide, ps = 0, 0, (0, 0)
    else:
        pos, wide = positions.data_ptr(), positions.dtype is torch.int64
        ps = positions.stride() if positions.shape[0] > 1 else (0, positions.stride(1))
    p = _params(dtype_code(q.dtype), b, s, d, hq, hk, q.data_ptr(), q_out.data_ptr(), kp, kop, *q.stride()[:3],
                *q_out.stride()[:3], *ks, *kos, turns.data_ptr(), 2 * turns.shape[0], interleaved, magnitude, inverse,
                pos, wide, *ps)
    _lib.run("attn_rotary", q.device, C.byref(p))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The gradient of a turn by +angle is a turn by -angle, and the other way round."""

    @staticmethod
    def forward(ctx, q, k, turns, positions, interleaved, magnitude, inverse):
        ctx.save_for_backward(turns, positions)
        ctx.how = interleaved, magnitude, inverse
        ctx.set_materialize_grads(False)
        out = _launch(q, k, turns, interleaved, magnitude, positions, inverse)
        return out if k is not None else out[0]

    @staticmethod
    def backward(ctx, gq, gk=None):
        turns, positions = ctx.saved_tensors
        interleaved, magnitude, inverse = ctx.how
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        if gq is not None and gk is not None:
            gq, gk = _turned(gq, gk, turns, positions, interleaved, magnitude, not inverse)
        elif gq is not None:
            gq = _turned(gq, None, turns, positions, interleaved, magnitude, not inverse)
        elif gk is not None:
            gk = _turned(gk, None, turns, positions, interleaved, magnitude, not inverse)
        return gq, gk, None, None, None, None, None


def _turned(q, k, *how):
    if differentiated(q, k):
        return _Rotary.apply(q, k, *how)
    turns, positions, interleaved, magnitude, inverse = how
    out = _launch(q, k, turns, interleaved, magnitude, positions, inverse)
    return out if k is not None else out[0]


_POSITIONS = (torch.int32, torch.int64)


def _fits(query, key, plan) -> bool:
    dev, dt, shape = query.device, query.dtype, query.shape
    if not (isinstance(plan, RotaryPlan) and plan.turns.device == dev and 2 * plan.turns.shape[0] <= shape[3]
            and plan.turns.dtype is torch.int64 and plan.turns.is_contiguous()):
        return False
    if key is None:
        return True
    return (isinstance(key, torch.Tensor) and key.dtype is dt and key.device == dev and key.dim() == 4
            and key.shape[0] == shape[0] and key.shape[2:] == shape[2:])


def _check(query, key, plan, positions):
    """Refuses what cannot be turned; the positions as the kernel reads them."""
    for name, x in (("query", query), ("key", key)):
        if x is None and name == "key":
            continue
        if not isinstance(x, torch.Tensor) or x.dim() != 4:
            raise ValueError(f"{name} must be (batch, heads, seq, head_dim)")
        dtype_code(x.dtype)
    b, _, s, d = query.shape
    if key is not None:
        if key.shape[0] != b or key.shape[2:] != query.shape[2:]:
            raise ValueError(f"key {tuple(key.shape)} does not match query {tuple(query.shape)}")
        if key.dtype != query.dtype:
            raise ValueError(f"key is {key.dtype}, query {query.dtype}")
        if key.device != query.device:
            raise RuntimeError("key must be on the query's device")
    check_plan(plan, d, query.device)
    if positions is not None:
        if not isinstance(positions, torch.Tensor):
            positions = torch.as_tensor(positions, device=query.device)
        if positions.is_floating_point() or positions.is_complex() or positions.dtype == torch.bool:
            raise ValueError(f"positions must be integers, got {positions.dtype}")
        if positions.dim() == 1:
            positions = positions[None]
        if positions.dim() != 2 or positions.shape[0] not in (1, b) or positions.shape[1] != s:
            raise ValueError(f"positions of shape {tuple(positions.shape)} do not match (B or 1, {s})")
        if positions.device != query.device:
            raise RuntimeError(f"positions must be on {query.device}")
        if positions.dtype not in (torch.int32, torch.int64):
            positions = positions.to(torch.int64)
    if not query.is_cuda:
        raise RuntimeError("attnax_b200 kernels need CUDA tensors; there is no CPU path")
    return positions


def apply_rotary(query: torch.Tensor, key: torch.Tensor | None, plan: RotaryPlan, *, positions=None,
                 inverse: bool = False):
    """Turns ``query (B, Hq, S, D)`` and ``key (B, Hkv, S, D)`` by their positions: ``(query', key')``; with ``key``
    ``None`` only ``query'``.  Differentiable (also twice).

    ``positions``: integers ``(S,)``, ``(1, S)`` or ``(B, S)`` on the tensors' device (default ``0 .. S-1``); they
    may be negative or of any size.  ``inverse=True`` turns backwards, which is the gradient (the plan's magnitude is
    a factor in both directions).  bf16, fp16 or fp32, any strides; each value
    is rounded once.  Results keep the inputs' dense layout (a transposed projection stays transposed).
    """
    # (one pass where all is well: the checks are a good part of a small call's host time)
    if not (isinstance(query, torch.Tensor) and query.is_cuda and query.dim() == 4 and _fits(query, key, plan)
            and (positions is None or (isinstance(positions, torch.Tensor) and positions.dim() == 2
                                       and positions.dtype in _POSITIONS and positions.device == query.device
                                       and positions.shape[0] in (1, query.shape[0])
                                       and positions.shape[1] == query.shape[2]))):
        positions = _check(query, key, plan, positions)
    how = (plan.turns, positions, plan.interleaved, plan.magnitude, bool(inverse))
    return _turned(query, key, *how)
