"""Rotary plans and the refusals of the rotary and 8-bit page operators (no GPU)."""

import ctypes
import dataclasses
import math
from fractions import Fraction

import pytest
import torch

import attnax_b200 as ax
from attnax_b200 import _lib, rotary


def test_frequencies_follow_their_formulas():
    n, r, base, length, f = 32, 64, 10000.0, 4096, 4.0
    w = [base ** (-i / n) for i in range(n)]

    def close(got, want):
        assert all(abs(g - x) <= 1e-14 * abs(x) for g, x in zip(got.tolist(), want))

    plain, m = ax.rotary_frequencies(r, base=base)
    close(plain, w)
    assert m == 1.0
    close(ax.rotary_frequencies(r, base=base, scaling="linear", factor=f)[0], [x / f for x in w])
    close(ax.rotary_frequencies(r, base=base, scaling="ntk", factor=f)[0],
          [(base * f ** (r / (r - 2))) ** (-i / n) for i in range(n)])
    got, m = ax.rotary_frequencies(r, base=base, scaling="yarn", factor=f, original_length=length)
    assert abs(m - (0.1 * math.log(f) + 1)) < 1e-15
    lo = math.floor(r * math.log(length / (2 * math.pi * 32)) / (2 * math.log(base)))
    hi = math.ceil(r * math.log(length / (2 * math.pi)) / (2 * math.log(base)))
    ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(n)]
    close(got, [x * (1 - g) + x / f * g for x, g in zip(w, ramp)])
    got, m = ax.rotary_frequencies(r, base=base, scaling="wavelength", factor=f, original_length=length)
    keep = [min(max((length * x / (2 * math.pi) - 1) / 3, 0.0), 1.0) for x in w]
    close(got, [x * k + x / f * (1 - k) for x, k in zip(w, keep)])
    assert keep[0] == 1.0 and keep[-1] == 0.0 and any(0 < k < 1 for k in keep)


@pytest.mark.parametrize("position", [0, 1, -1, 4095, 1_000_003, 2**31 - 1, -2**31, 2**40 + 12345])
def test_plan_holds_angles_at_any_position(position):
    w, _ = ax.rotary_frequencies(64)
    plan = ax.rotary_plan(64, device="cpu")
    for x, bits in zip(w.tolist(), plan.turns.tolist()):
        turn = Fraction(x / (2 * math.pi))  # the 64-bit quotient that the plan starts from
        want = (turn * position) % 1
        got = Fraction((bits * position) % 2**64, 2**64)
        off = abs(want - got)
        assert min(off, 1 - off) <= Fraction(abs(position) + 1, 2**64)


def test_plan_takes_frequencies_of_any_sign_and_size():
    plan = ax.rotary_plan_from_frequencies([2 * math.pi * 0.25, -2 * math.pi * 0.25, 2 * math.pi * 3.5], device="cpu")
    got = [b % 2**64 / 2**64 for b in plan.turns.tolist()]
    assert got == pytest.approx([0.25, 0.75, 0.5], abs=1e-15)
    assert plan.rotary_dim == 6


@pytest.mark.parametrize("kw", [
    {"rotary_dim": 0}, {"rotary_dim": 7}, {"rotary_dim": -2}, {"rotary_dim": 8, "base": 0.0},
    {"rotary_dim": 8, "factor": 2.0}, {"rotary_dim": 8, "scaling": "other"},
    {"rotary_dim": 8, "scaling": "linear", "factor": 0.0}, {"rotary_dim": 2, "scaling": "ntk", "factor": 2.0},
    {"rotary_dim": 8, "scaling": "yarn", "factor": 2.0}, {"rotary_dim": 8, "scaling": "wavelength", "factor": 2.0},
    {"rotary_dim": 8, "scaling": "yarn", "factor": 2.0, "original_length": 10, "beta_fast": 1.0, "beta_slow": 2.0},
    {"rotary_dim": 8, "scaling": "wavelength", "factor": 2.0, "original_length": 10, "low_factor": 4.0},
    {"rotary_dim": 8, "scaling": "linear", "factor": float("nan")},
])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        ax.rotary_plan(device="cpu", **kw)


def test_plan_from_frequencies_refusals():
    for bad in ([], [[1.0]], [float("inf")], [float("nan"), 1.0]):
        with pytest.raises(ValueError):
            ax.rotary_plan_from_frequencies(bad, device="cpu")


def test_apply_rotary_refusals():
    plan = ax.rotary_plan(8, device="cpu")
    q, k = torch.zeros(2, 4, 5, 8), torch.zeros(2, 2, 5, 8)
    for args, kw in [
        ((q[0], None, plan), {}), ((q, k[0], plan), {}), ((q.int(), None, plan), {}), ((q, k.half(), plan), {}),
        ((q, k[:1], plan), {}), ((q, k[:, :, :4], plan), {}), ((q[..., :6], None, plan), {}), ((q, k, None), {}),
        ((q, k, plan), {"positions": torch.zeros(5)}), ((q, k, plan), {"positions": torch.zeros(4, dtype=torch.int32)}),
        ((q, k, plan), {"positions": torch.zeros(3, 5, dtype=torch.int32)}),
        ((q, k, plan), {"positions": torch.zeros(1, 1, 5, dtype=torch.int32)}),
    ]:
        with pytest.raises(ValueError):
            ax.apply_rotary(*args, **kw)
    with pytest.raises(RuntimeError):
        ax.apply_rotary(q, k, plan)  # no CPU path


def _cache(dtype=torch.int8, **kw):
    shape = dict(num_blocks=4, block_size=16, num_kv_heads=2, head_dim=8, batch_size=2, max_blocks_per_seq=2) | kw
    if dtype in (torch.int8, torch.float8_e4m3fn):
        return ax.init_quantized_paged_kv_cache(**shape, dtype=dtype, device="cpu")
    return ax.init_paged_kv_cache(**shape, dtype=dtype, device="cpu")


def _with(cache, **kw):
    import dataclasses
    return dataclasses.replace(cache, **kw)


def test_quantized_cache_shapes():
    c = _cache(torch.float8_e4m3fn)
    assert (c.num_blocks, c.block_size, c.num_kv_heads, c.head_dim) == (4, 16, 2, 8)
    assert c.key_scales.shape == (4, 2) and bool((c.key_scales == 1).all())
    assert bool((c.block_table == -1).all()) and bool((c.seq_lengths == 0).all())
    with pytest.raises(ValueError):
        ax.init_quantized_paged_kv_cache(num_blocks=4, block_size=16, num_kv_heads=2, head_dim=8, batch_size=2,
                                         max_blocks_per_seq=2, dtype=torch.float8_e5m2, device="cpu")


def test_cache_refusals():
    good, k = _cache(), torch.zeros(2, 2, 3, 8)
    q = torch.zeros(2, 4, 1, 8)
    for bad, err in [
        (_with(good, key_scales=good.key_scales[:3]), ValueError),
        (_with(good, value_scales=good.value_scales.double()), ValueError),
        (_with(good, value_scales=good.value_scales.T.contiguous().T), ValueError),
        (_with(good, value_pool=good.value_pool[:, :, :1]), ValueError),
        (_with(good, key_pool=good.key_pool.float(), value_pool=good.value_pool.float()), ValueError),
        (_with(good, block_table=good.block_table.long()), ValueError),
        (_with(good, seq_lengths=good.seq_lengths[:1]), ValueError),
        (_with(good, key_pool=good.key_pool.transpose(1, 2), value_pool=good.value_pool.transpose(1, 2)), ValueError),
        ("cache", ValueError),
    ]:
        with pytest.raises(err):
            ax.append_tokens(bad, k, k)
        with pytest.raises(err):
            ax.gather_tokens(bad, None, 3)
        with pytest.raises(err):
            ax.paged_quantized_attention(q, bad)
    with pytest.raises(ValueError):
        ax.paged_quantized_attention(q, _cache(torch.bfloat16))
    # a cache of the other kind is not taken for a 16-bit one
    with pytest.raises(ValueError):
        ax.paged_attention_batched(q, good)


def test_append_and_gather_refusals():
    c, k = _cache(), torch.zeros(2, 2, 3, 8)
    plan = ax.rotary_plan(8, device="cpu")
    for args, kw in [
        ((k[0], k[0]), {}), ((k[:1], k[:1]), {}), ((k[:, :1], k[:, :1]), {}), ((k[..., :4], k[..., :4]), {}),
        ((k, k[:, :, :2]), {}), ((k, k.half()), {}), ((k.int(), k.int()), {}),
        ((k, k), {"query": torch.zeros(2, 4, 3, 8)}),  # nothing to turn it by
        ((k, k), {"query": torch.zeros(2, 4, 2, 8), "rotary": plan}),
        ((k, k), {"query": torch.zeros(2, 4, 3, 8).half(), "rotary": plan}),
        ((k, k), {"rotary": ax.rotary_plan(10, device="cpu")}), ((k, k), {"rotary": "plan"}),
    ]:
        with pytest.raises(ValueError):
            ax.append_tokens(c, *args, **kw)
    with pytest.raises(RuntimeError):
        ax.append_tokens(c, k, k)
    with pytest.raises(ValueError):
        ax.gather_tokens(c, None, -1)
    with pytest.raises(ValueError):
        ax.gather_tokens(c, torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(ValueError):
        ax.gather_tokens(c, None, 2, dtype=torch.int8)
    with pytest.raises(RuntimeError):
        ax.gather_tokens(c, None, 2)


def test_attention_refusals():
    c = _cache()
    for q in (torch.zeros(2, 4, 8), torch.zeros(1, 4, 1, 8), torch.zeros(2, 3, 1, 8), torch.zeros(2, 4, 1, 16),
              torch.zeros(2, 4, 1, 8, dtype=torch.int8)):
        with pytest.raises(ValueError):
            ax.paged_quantized_attention(q, c)
    with pytest.raises(RuntimeError):
        ax.paged_quantized_attention(torch.zeros(2, 4, 1, 8), c)


def test_taylor_borders():
    """The kernel's series leave less than half a step of fp32 at the border of a quarter turn's half."""
    x = math.pi / 4
    assert x ** 11 / math.factorial(11) < 2.0 ** -25 * math.sin(x)
    assert x ** 12 / math.factorial(12) < 2.0 ** -25 * math.cos(x)
    assert rotary.RotaryPlan is ax.RotaryPlan


def test_struct_layouts_match_the_c_compiler(tmp_path):
    """Offsets and sizes of the ctypes mirrors equal what gcc computes from the header."""
    import ctypes
    import pathlib
    import shutil
    import subprocess

    from attnax_b200 import _lib

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    root = pathlib.Path(__file__).resolve().parent.parent
    structs = {"attn_rotary_spec_t": _lib.RotarySpec, "attn_rotary_params_t": _lib.RotaryParams,
               "attn_paged_append_params_t": _lib.PagedAppendParams,
               "attn_paged_gather_params_t": _lib.PagedGatherParams,
               "attn_paged_attend8_params_t": _lib.PagedAttend8Params}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{root}/include/attnb200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'printf("{cname}.{fname} %zu\\n", offsetof({cname}, {fname}));')
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", tmp_path / "layout", tmp_path / "layout.c"], check=True)
    got = dict(x.split() for x in subprocess.run([tmp_path / "layout"], check=True, capture_output=True,
                                                 text=True).stdout.splitlines())
    for cname, py in structs.items():
        assert int(got[cname]) == ctypes.sizeof(py), cname
        for fname, _ in py._fields_:
            assert int(got[f"{cname}.{fname}"]) == getattr(py, fname).offset, f"{cname}.{fname}"


def test_strided_pools_of_other_types_are_still_gathered():
    """gather_kv reads pools that no kernel can address through torch, whatever their type."""
    for dt in (torch.float64, torch.int8):
        pool = torch.arange(4 * 16 * 2 * 8, dtype=torch.int64).remainder(100).to(dt).view(4, 2, 16, 8).transpose(1, 2)
        cache = ax.PagedKVCache(pool, pool, torch.tensor([[2, 1]], dtype=torch.int32),
                                torch.tensor([20], dtype=torch.int32))
        k, v, n = ax.gather_kv(cache, 0)
        want = torch.cat([pool[2], pool[1]])[:20]
        assert n == 20 and torch.equal(k, want) and torch.equal(v, want)


def test_codes_are_not_taken_for_values():
    cache = ax.init_quantized_paged_kv_cache(num_blocks=4, block_size=16, num_kv_heads=2, head_dim=8, batch_size=1,
                                             max_blocks_per_seq=2, device="cpu")
    for c in (cache, dataclasses.replace(cache, key_pool=cache.key_pool.transpose(1, 2).contiguous().transpose(1, 2),
                                         value_pool=cache.value_pool.transpose(1, 2).contiguous().transpose(1, 2))):
        for call in (lambda: ax.gather_kv(c, 0),
                     lambda: ax.append_kv(c, 0, torch.zeros(1, 2, 8), torch.zeros(1, 2, 8)),
                     lambda: ax.paged_attention(torch.zeros(2, 1, 8), c, 0)):
            with pytest.raises(ValueError, match="codes"):
                call()
    wide = dataclasses.replace(cache, block_table=cache.block_table.long())
    with pytest.raises(ValueError, match="block_table"):
        ax.append_tokens(wide, torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8))


def test_pages_whose_offsets_pass_32_bits_are_refused():
    """Refused on the host, before anything is read through the pointers (which are never followed)."""
    x = torch.zeros(64, dtype=torch.int64)
    p = _lib.PagedAppendParams()
    p.dtype, p.pool_format, p.num_blocks = _lib.ATTN_BF16, _lib.POOL_E4M3, 1
    p.block_size, p.num_heads_kv, p.head_dim = 1 << 20, 64, 64
    p.num_seqs, p.max_blocks_per_seq, p.num_new = 1, 1, 1
    for name in ("key_pool", "value_pool", "key_scales", "value_scales", "block_table", "seq_lengths", "keys", "values",
                 "lengths_out"):
        setattr(p, name, x.data_ptr())
    status = _lib.load().attn_paged_append_tokens(ctypes.byref(p), None)
    with pytest.raises(NotImplementedError):
        _lib.check(status, "attn_paged_append_tokens")
