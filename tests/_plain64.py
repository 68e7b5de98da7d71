"""Plain attention in 64 bits and the rounding bounds that the operator tests hold the kernels to."""

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Smallest rounding step of the type itself: what a value below its normal range is off by at most.
TINY_STEP = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
MEAN_REL = 1e-2  # the framework's bar for 16-bit outputs (mean relative error)


def softmax_rows(x, keep):
    """Softmax over the kept columns in x's type; rows that keep nothing are zero."""
    x = x.masked_fill(~keep, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    s = p.sum(-1, keepdim=True)
    return p / torch.where(s == 0, torch.ones_like(s), s)


def attention64(q, k, v, keep, do=None, bias=None):
    """(out, bound[, grads, bounds]) of softmax(q k^T / sqrt(D) + bias | keep) v in 64 bits.

    q (B, Hq, T, D), k/v (B, Hkv, N, D) in the kernels' type; keep broadcasts to
    (B, Hq, T, N).  ``bound`` is how far a kernel that works in 32 bits and
    rounds P (and dS) once to the inputs' type may be off per element.
    """
    dt = q.dtype
    h, tiny = HALF_STEP[dt], TINY_STEP[dt]
    grp = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(grp, 1), v.double().repeat_interleave(grp, 1)
    d = q.shape[-1]
    sc = 1.0 / math.sqrt(d)
    x = q @ k.transpose(-1, -2) * sc
    if bias is not None:
        x = x + bias
    p = softmax_rows(x, keep)
    out = p @ v
    # A score is a sum of d products held in 32 bits (and one bias), so the exponent is off by at
    # most (d + 4) half steps of the sum of magnitudes; the exponential and the row sum (n terms,
    # added in any order) add a relative error of a few steps.  Both sides of P = e / l carry it.
    mag = float((q.abs() @ k.abs().transpose(-1, -2)).amax()) * sc
    if bias is not None:
        mag += float(bias.abs().amax())
    n = k.shape[2]
    rel = 2 * ((d + 4) * 2.0 ** -24 * mag + 2.0 ** -20) + math.sqrt(n) * 2.0 ** -22
    pv = p @ v.abs()
    bound = (h + rel) * pv + h * out.abs() + tiny * (v.abs().sum(-2, keepdim=True) + 1) + 1e-30
    if do is None:
        return out, bound
    do = do.double()
    dp = do @ v.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # delta comes from the rounded output; dP and delta are sums held in 32 bits
    d_delta = (do.abs() * bound).sum(-1, keepdim=True)
    dp_mag = do.abs() @ v.abs().transpose(-1, -2)
    e_ds = (h + rel) * ds.abs() + p * (d_delta + rel * (dp_mag + delta.abs())) + tiny
    e_p = (h + rel) * p + tiny
    B, Hq = q.shape[:2]

    def fold(t):
        return t.view(B, Hq // grp, grp, *t.shape[2:]).sum(2)

    dq = ds @ k * sc
    dk = fold(ds.transpose(-1, -2) @ q) * sc
    dv = fold(p.transpose(-1, -2) @ do)
    # the sums of the gradients themselves run in 32 bits over up to T * grp terms
    acc = math.sqrt(max(n, q.shape[2] * grp)) * 2.0 ** -22
    bq = (e_ds + acc * ds.abs()) @ k.abs() * sc + h * dq.abs() + tiny
    bk = fold((e_ds + acc * ds.abs()).transpose(-1, -2) @ q.abs()) * sc + h * dk.abs() + tiny
    bv = fold((e_p + acc * p).transpose(-1, -2) @ do.abs()) + h * dv.abs() + tiny
    return out, bound, (dq, dk, dv), (bq, bk, bv)


def assert_within(got, want, bound, what=""):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    err = (got - want).abs()
    worst = float((err / bound).amax()) if err.numel() else 0.0
    total = float(want.abs().sum())
    rel = float(err.sum()) / total if total else 0.0
    print(f"[plain64] {what}: worst error / bound {worst:.3f}, mean-rel {rel:.2e}")
    assert worst <= 1.0, f"{what}: an element is {worst:.3f} times its bound off"
    # A relative error says nothing of values that are smaller than what they may be off by: with a
    # single visible key P = 1 and dS = dP - delta is 0, but dP and delta are sums of D products in 32
    # bits in two orders, each off by up to D 2^-24 of the sum of magnitudes (the bound above).
    if total < float(bound.expand_as(want).sum()):
        return
    assert rel <= MEAN_REL, f"{what}: mean relative error {rel:.3e}"
