"""Workloads of the rotary positions, of tokens appended to paged caches, and of attention over 8-bit pages.

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the same ranges;
``prepare`` makes what a program holds before the call, ``run`` is one call of
an operator (its plain form in elementary torch operations, or this package's
kernels when ``own`` is set), ``exact`` the same outputs from the definitions
in 64 bits, and ``work`` the bytes and operations one call cannot do without.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
          "int8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # One decode step of a serving batch: 64 sequences, a token each, every one at its own position.
        {"name": "rotary_decode_b64", "kind": "rotary", "dtype": "bf16", "batch": 64, "heads": 32, "kv_heads": 8,
         "seq": 1, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "wavelength", "factor": 8.0,
         "first": 100000, "train": False},
        # Training at the benchmarked shape with positions stretched for long contexts: both tensors, both directions.
        {"name": "rotary_train_bf16_s8192", "kind": "rotary", "dtype": "bf16", "batch": 4, "heads": 32, "kv_heads": 8,
         "seq": 8192, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "yarn", "factor": 4.0, "first": 0,
         "train": True},
        # Neighbouring pairs, a part of the head only, odd length, heads not a power of two, positions far out.
        {"name": "rotary_train_f16_part", "kind": "rotary", "dtype": "f16", "batch": 3, "heads": 12, "kv_heads": 4,
         "seq": 1999, "dim": 64, "rotary": 32, "interleaved": True, "scaling": "ntk", "factor": 2.0,
         "first": 1000000, "train": True},
        # The fp32 path at the shape that the parity tests train.
        {"name": "rotary_train_f32", "kind": "rotary", "dtype": "f32", "batch": 2, "heads": 8, "kv_heads": 8,
         "seq": 1024, "dim": 64, "rotary": 64, "interleaved": False, "scaling": "none", "factor": 1.0, "first": 0,
         "train": True},
        # A decode step into a 16-bit cache: keys and queries rotated on the way.
        {"name": "append_decode_bf16", "kind": "append", "dtype": "bf16", "pool": "bf16", "batch": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "page": 16, "ctx_lo": 512, "ctx_hi": 4096,
         "tokens": 1},
        # Prompts of different lengths, padded, go into the cache at once; some continue a prefix.
        {"name": "append_prompt_bf16", "kind": "append", "dtype": "bf16", "pool": "bf16", "batch": 8, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "page": 16, "ctx_lo": 0, "ctx_hi": 1000,
         "tokens": 4096},
        # A decode step into 8-bit pages: a page whose scale grows is restated.
        {"name": "append_decode_e4m3", "kind": "append", "dtype": "bf16", "pool": "e4m3", "batch": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "page": 16, "ctx_lo": 512, "ctx_hi": 32768,
         "tokens": 1},
        # Prompts into 8-bit pages of integers, half of the head rotated, fp16 model with larger pages.
        {"name": "append_prompt_int8", "kind": "append", "dtype": "f16", "pool": "int8", "batch": 8, "heads": 16,
         "kv_heads": 8, "dim": 128, "rotary": 64, "interleaved": True, "page": 64, "ctx_lo": 0, "ctx_hi": 777,
         "tokens": 4001},
        # One token of one reply over 8-bit pages, where latency counts.
        {"name": "attend_e4m3_b1", "kind": "attend", "dtype": "bf16", "pool": "e4m3", "batch": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "ctx_lo": 2500, "ctx_hi": 2500, "tokens": 1},
        # The serving batch of the paged decode benchmark, in 8 bits.
        {"name": "attend_e4m3_b64", "kind": "attend", "dtype": "bf16", "pool": "e4m3", "batch": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "ctx_lo": 512, "ctx_hi": 32768, "tokens": 1},
        # A few tokens per sequence (a verified draft), integers, head dim 64, odd batch, fp16.
        {"name": "attend_int8_t5", "kind": "attend", "dtype": "f16", "pool": "int8", "batch": 13, "heads": 12,
         "kv_heads": 4, "dim": 64, "page": 32, "ctx_lo": 300, "ctx_hi": 20011, "tokens": 5},
        # A chunk of a prompt against the pages before it.
        {"name": "attend_e4m3_t64", "kind": "attend", "dtype": "bf16", "pool": "e4m3", "batch": 8, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "ctx_lo": 1000, "ctx_hi": 16384, "tokens": 64},
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend"])
    half = rng.choice(["bf16", "bf16", "f16"])
    kvh = rng.choice([1, 2, 4, 8])
    heads = kvh * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128])
        dtype = rng.choice([half, half, "f32"])
        return {"kind": kind, "dtype": dtype, "batch": rng.choice([1, 2, 3, 4]), "heads": min(heads, 32),
                "kv_heads": kvh, "seq": _logint(rng, 1, 4096 if dtype == "f32" else 8192), "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                "factor": rng.choice([1.5, 2.0, 4.0, 8.0]), "first": rng.choice([0, rng.randrange(1000000)]),
                "train": rng.random() < 0.6}
    pool = rng.choice(["e4m3", "int8"])
    if kind == "append":
        return {"kind": kind, "dtype": half, "pool": rng.choice([pool, pool, half]), "batch": rng.randrange(1, 33),
                "heads": min(heads, 32), "kv_heads": kvh, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
                "interleaved": rng.random() < 0.5, "page": page, "ctx_lo": rng.choice([0, 37]),
                "ctx_hi": _logint(rng, 64, 4096), "tokens": rng.choice([1, _logint(rng, 1, 1024)])}
    tokens = rng.choice([1, 1, rng.randrange(2, 9), rng.randrange(9, 65)])
    hi = _logint(rng, 64, 16384 if tokens > 8 else 32768)
    return {"kind": kind, "dtype": half, "pool": pool, "batch": _logint(rng, 1, 8 if tokens > 8 else 48),
            "heads": min(heads, 32), "kv_heads": kvh, "dim": dim, "page": page, "ctx_lo": max(1, hi // 50),
            "ctx_hi": hi, "tokens": tokens}


# ------------------------------------------------------------------ numbers --
# Original context of the stretched positions, and the borders of the scaled forms (the usual ones).
ORIGINAL, FAST, SLOW, LOW, HIGH = 4096, 32.0, 1.0, 1.0, 4.0
BASE = 10000.0


def _frequencies(rotary, scaling, factor):
    """(radians per position of each pair, in 64 bits on the host; the factor on both tensors)."""
    n = rotary // 2
    i = torch.arange(n, dtype=torch.float64)
    base = BASE * factor ** (rotary / (rotary - 2)) if scaling == "ntk" else BASE
    w = base ** (-i / n)
    if scaling == "linear":
        return w / factor, 1.0
    if scaling == "yarn":
        def at(turns):
            return rotary * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(BASE))

        lo, hi = max(math.floor(at(FAST)), 0), min(math.ceil(at(SLOW)), rotary - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w * (1 - ramp) + w / factor * ramp, 0.1 * math.log(factor) + 1
    if scaling == "wavelength":
        keep = ((ORIGINAL * w / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        return w * keep + w / factor * (1 - keep), 1.0
    return w, 1.0


def _case_frequencies(case):
    return _frequencies(case["rotary"], case.get("scaling", "none"), case.get("factor", 1.0))


def _lengths(case):
    """Context lengths spread evenly over the logarithm of the case's range, in a mixed order; they are part of the case."""
    lo, hi, b = max(case["ctx_lo"], 1), case["ctx_hi"], case["batch"]
    at = [0.5 if b == 1 else ((i * 0.6180339887498949) % 1.0) for i in range(b)]
    n = [int(round(math.exp(math.log(lo) + x * (math.log(hi) - math.log(lo))))) for x in at]
    if case["ctx_lo"] == 0:
        n = [0 if i % 3 == 0 else x for i, x in enumerate(n)]
    return n


def _new_lengths(case):
    """Tokens that each sequence appends: all of them in a decode step, a padded batch otherwise (one of it may have none)."""
    t, b = case["tokens"], case["batch"]
    if t == 1:
        return [1] * b
    return [t if i == 0 else int(t * ((i * 0.7548776662466927) % 1.0)) for i in range(b)]


def _pool_scale(amax, pool):
    """The least power of two, 2^-100 at least, that brings ``amax`` into the 8-bit type."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8) if pool == "e4m3" else torch.where(m <= 127 / 128, e - 7, e - 6)
    k = torch.where(amax == 0, torch.full_like(k, -100), k.clamp(min=-100))
    return torch.ldexp(torch.ones_like(amax), k)


def _to_bits(x, pool):
    return x.to(torch.float8_e4m3fn) if pool == "e4m3" else x.round().to(torch.int8)


# ----------------------------------------------------------------- prepare --
def _gens(seed):
    c = torch.Generator()
    c.manual_seed(seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return c, g


def _randn(g, shape, dt):
    return torch.randn(shape, generator=g, device=DEV, dtype=dt)


def _token_rows(g, shape, dt, keys):
    """Projected tokens; keys have a few channels that are several times as large as the others."""
    x = _randn(g, shape, dt)
    if keys:
        x[..., 5::37] *= 6
    return x


def _pages(case, lens, c, g):
    """Pools of random pages and the table; an 8-bit pool holds tokens that were brought to 8 bits page by page."""
    bs, hk, d, pool = case["page"], case["kv_heads"], case["dim"], case["pool"]
    need = [-(-n // bs) for n in lens]
    nb, most = sum(need) + 3, max(max(need), 1)
    perm = torch.randperm(nb, generator=c).to(torch.int32)
    table = torch.full((len(lens), most), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    st = {"table": table.to(DEV)}
    for name in ("k", "v"):
        if SIZE[pool] > 1:
            st[name] = _token_rows(g, (nb, bs, hk, d), DTYPES[pool], name == "k")
            continue
        codes = torch.empty((nb, bs, hk, d), dtype=DTYPES[pool], device=DEV)
        scales = torch.empty((nb, hk), dtype=torch.float32, device=DEV)
        for b0 in range(0, nb, 4096):
            x = _token_rows(g, (min(4096, nb - b0), bs, hk, d), torch.float32, name == "k")
            s = _pool_scale(x.abs().amax((1, 3)), pool)
            codes[b0:b0 + 4096] = _to_bits(x / s[:, None, :, None], pool)
            scales[b0:b0 + 4096] = s
        st[name], st[name + "_scales"] = codes, scales
    return st


def prepare(case, seed):
    c, g = _gens(seed)
    kind, dt, d = case["kind"], DTYPES[case["dtype"]], case["dim"]
    b, h, hk = case["batch"], case["heads"], case["kv_heads"]
    st = {"case": case}
    if kind == "rotary":
        s = case["seq"]
        # the projections' layout: (batch, tokens, heads, dim), seen as (batch, heads, tokens, dim)
        for name, n in (("q", h), ("k", hk)):
            st[name] = _randn(g, (b, s, n, d), dt).transpose(1, 2).requires_grad_(case["train"])
            if case["train"]:
                st["d" + name] = _randn(g, (b, n, s, d), dt)
        first = torch.randint(0, case["first"] + 1, (b, 1), generator=c)
        st["positions"] = (first + torch.arange(s)).to(torch.int32).to(DEV)
        w, st["magnitude"] = _case_frequencies(case)
        st["frequencies"] = w.to(DEV)
        if own:
            import attnax_b200 as ax

            kw = {} if case["scaling"] == "none" else {"scaling": case["scaling"], "factor": case["factor"],
                                                      "original_length": ORIGINAL}
            st["plan"] = ax.rotary_plan(case["rotary"], base=BASE, interleaved=case["interleaved"], device=DEV, **kw)
        return st
    lens = _lengths(case)
    if kind == "append":
        t, new = case["tokens"], _new_lengths(case)
        st.update(_pages(case, [x + y for x, y in zip(lens, new)], c, g))
        st["q"] = _randn(g, (b, t, h, d), dt).transpose(1, 2)
        st["new_k"] = _token_rows(g, (b, t, hk, d), dt, True).transpose(1, 2)
        st["new_v"] = _token_rows(g, (b, t, hk, d), dt, False).transpose(1, 2)
        st["new_lens"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        st["starts"] = torch.tensor([x // case["page"] * case["page"] for x in lens], dtype=torch.int32, device=DEV)
        st["frequencies"] = _case_frequencies(case)[0].to(DEV)
    else:
        lens = [max(n, case["tokens"]) for n in lens]
        st.update(_pages(case, lens, c, g))
        st["q"] = _randn(g, (b, h, case["tokens"], d), dt)
        st["max_ctx"] = max(lens)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if own:
        import attnax_b200 as ax

        if kind == "append":
            st["plan"] = ax.rotary_plan(case["rotary"], base=BASE, interleaved=case["interleaved"], device=DEV)
        if SIZE[case["pool"]] == 1:
            st["cache"] = ax.QuantizedPagedKVCache(st["k"], st["v"], st["k_scales"], st["v_scales"], st["table"],
                                                   st["lens"])
        else:
            st["cache"] = ax.PagedKVCache(st["k"], st["v"], st["table"], st["lens"])
    return st


# --------------------------------------------------------------- plain forms --
def _turned(x, cos, sin, case):
    """``x (..., dim)`` in 32 bits with its first ``rotary`` channels turned; cos and sin hold a value per pair."""
    r = case["rotary"]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., r:]], -1) if r < x.shape[-1] else y


def _cos_sin(positions, frequencies, magnitude=1.0):
    """(batch, 1, tokens, pairs), the angles in 64 bits: 32 lose whole radians of far positions."""
    angle = (positions[..., None].double() * frequencies)[:, None]
    return (magnitude * torch.cos(angle)).float(), (magnitude * torch.sin(angle)).float()


def _plain_rotary(st):
    case = st["case"]
    cos, sin = _cos_sin(st["positions"], st["frequencies"], st["magnitude"])
    dt = st["q"].dtype
    out = {}
    for name in ("q", "k"):
        out[name] = _turned(st[name].detach().float(), cos, sin, case).to(dt)
        if case["train"]:
            out["d" + name] = _turned(st["d" + name].float(), cos, -sin, case).to(dt)
    return out


def _slots(st, tokens):
    """For the new tokens: (whether each is there, its position)."""
    i = torch.arange(tokens, device=DEV)
    return i < st["new_lens"][:, None], st["lens"][:, None] + i


def _plain_append(st):
    case = st["case"]
    bs, hk, d, t, pool = case["page"], case["kv_heads"], case["dim"], case["tokens"], case["pool"]
    there, pos = _slots(st, t)
    cos, sin = _cos_sin(pos, st["frequencies"])
    q = _turned(st["q"].float(), cos, sin, case).to(st["q"].dtype)
    rows = {"k": _turned(st["new_k"].float(), cos, sin, case).transpose(1, 2),
            "v": st["new_v"].float().transpose(1, 2)}  # (batch, tokens, kv heads, dim)
    lens = st["lens"] + st["new_lens"]
    page = st["table"].long().gather(1, (pos // bs).clamp(max=st["table"].shape[1] - 1))
    if SIZE[pool] > 1:
        at = (page * bs + pos % bs)[there]
        for name in ("k", "v"):
            st[name].view(-1, hk, d)[at] = rows[name][there].to(st[name].dtype)
        return {"q": q, "k": st["k"], "v": st["v"], "lens": lens}
    # 8 bits: the pages from the first that the call touches on, token by token
    width = -(-(t + bs - 1) // bs) * bs
    j = torch.arange(width, device=DEV)
    at = st["starts"][:, None] + j
    old, new = at < st["lens"][:, None], (at >= st["lens"][:, None]) & (at < lens[:, None])
    touched = new.view(-1, width // bs, bs).any(-1)
    ids = st["table"].long().gather(1, (at[:, ::bs] // bs).clamp(max=st["table"].shape[1] - 1)).clamp(min=0)
    src = (at - st["lens"][:, None]).clamp(0, t - 1)
    out = {"q": q, "lens": lens}
    for name in ("k", "v"):
        x = rows[name].gather(1, src[:, :, None, None].expand(-1, -1, hk, d)) * new[:, :, None, None]
        had = old.view(-1, width // bs, bs).any(-1)
        s_old = st[name + "_scales"][ids] * had[:, :, None]
        codes = st[name].view(torch.uint8)[ids].view(st[name].dtype).float()  # (batch, pages, page, kv heads, dim)
        x = x.view(codes.shape)
        s = torch.maximum(s_old, _pool_scale(x.abs().amax((2, 4)), pool))
        both = torch.where(old.view(-1, width // bs, bs)[..., None, None], codes * (s_old / s)[:, :, None, :, None],
                           x / s[:, :, None, :, None])
        both = _to_bits(both, pool)
        w = touched
        st[name].view(torch.uint8)[ids[w]] = both.view(torch.uint8)[w]
        st[name + "_scales"][ids[w]] = s[w]
        now = st[name].view(torch.uint8)[ids].view(st[name].dtype).float() * st[name + "_scales"][ids][:, :, None, :, None]
        now = now * (old | new).view(-1, width // bs, bs)[..., None, None]
        out[name] = now.reshape(-1, width, hk, d).transpose(1, 2).to(q.dtype)
    return out


def _plain_attend(st):
    case = st["case"]
    q, hk, d, t = st["q"], case["kv_heads"], case["dim"], case["tokens"]
    b, h = q.shape[:2]
    ids = st["table"].long().clamp(min=0)
    n = ids.shape[1] * case["page"]

    def held(name):  # (batch, kv heads, tokens, dim)
        x = st[name].view(torch.uint8)[ids].view(st[name].dtype).float()
        return x.mul_(st[name + "_scales"][ids][:, :, None, :, None]).view(b, n, hk, d).transpose(1, 2)

    x = (q.float() / math.sqrt(d)).view(b, hk, (h // hk) * t, d) @ held("k").transpose(2, 3)
    last = (st["lens"][:, None] - t + torch.arange(t, device=DEV)).repeat(1, h // hk)  # each row's position
    x = x.masked_fill_((torch.arange(n, device=DEV) > last[:, :, None])[:, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = (p @ held("v")) / p.sum(-1, keepdim=True)
    return {"out": o.view(b, h, t, d).to(q.dtype)}


# --------------------------------------------------------------------- run --
def _own(st):
    import attnax_b200 as ax

    case = st["case"]
    if case["kind"] == "rotary":
        q, k = ax.apply_rotary(st["q"], st["k"], st["plan"], positions=st["positions"])
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["kind"] == "attend":
        return {"out": ax.paged_quantized_attention(st["q"], st["cache"], max_context=st["max_ctx"])}
    cache, q = ax.append_tokens(st["cache"], st["new_k"], st["new_v"], new_lengths=st["new_lens"],
                                rotary=st["plan"], query=st["q"], check=False)
    if SIZE[case["pool"]] > 1:
        return {"q": q, "k": cache.key_pool, "v": cache.value_pool, "lens": cache.seq_lengths}
    width = -(-(case["tokens"] + case["page"] - 1) // case["page"]) * case["page"]
    k, v = ax.gather_tokens(cache, st["starts"], width, dtype=q.dtype)
    return {"q": q, "k": k, "v": v, "lens": cache.seq_lengths}


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- exact --
def _exact_turn(x, positions, w, interleaved, sign=1.0, magnitude=1.0):
    """Pairs as complex numbers times e^(i angle), in 64 bits; ``x (batch, heads, tokens, dim)``."""
    n = w.numel()
    x = x.detach().double().clone()
    first = x[..., 0:2 * n:2] if interleaved else x[..., :n]
    second = x[..., 1:2 * n:2] if interleaved else x[..., n:2 * n]
    angle = sign * positions.double()[:, None, :, None] * w
    z = torch.complex(first, second) * torch.polar(torch.full_like(angle, magnitude), angle)
    if interleaved:
        x[..., 0:2 * n:2], x[..., 1:2 * n:2] = z.real, z.imag
    else:
        x[..., :n], x[..., n:2 * n] = z.real, z.imag
    return x


def _exact_round(y, pool):
    """The nearest value of the 8-bit type (even ones at ties), from its steps."""
    if pool == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_page(page, old, old_scale, pool):
    """Values ``(tokens, kv heads, dim)`` of an 8-bit page, the first ``old`` of them codes of ``old_scale (kv heads)``."""
    most = {"e4m3": 448.0, "int8": 127.0}[pool]
    amax = page[old:].abs().amax((0, 2))
    s = torch.ldexp(torch.ones_like(amax), (torch.round(torch.log2(amax / most)) + 1).int())  # one or two steps too large
    s = torch.where(amax <= most * s / 4, s / 4, torch.where(amax <= most * s / 2, s / 2, s)).clamp(min=2.0 ** -100)
    s = torch.maximum(s, old_scale)[:, None]
    return torch.cat([_exact_round(page[:old] * (old_scale[:, None] / s), pool), _exact_round(page[old:] / s, pool)]) * s


def _exact_append(st):
    """Tokens that were there before are restated where their page's scale grows."""
    case = st["case"]
    bs, hk, d, t, b = case["page"], case["kv_heads"], case["dim"], case["tokens"], case["batch"]
    w = _case_frequencies(case)[0].to(DEV)
    pos = st["lens"].long()[:, None] + torch.arange(t, device=DEV)
    q = _exact_turn(st["q"], pos, w, case["interleaved"])
    new = {"k": _exact_turn(st["new_k"], pos, w, case["interleaved"]), "v": st["new_v"].double()}
    lens, counts, starts = st["lens"].tolist(), st["new_lens"].tolist(), st["starts"].tolist()
    wide = SIZE[case["pool"]] > 1
    width = -(-(t + bs - 1) // bs) * bs
    out = {"q": q, "lens": st["lens"] + st["new_lens"]}
    for name in ("k", "v"):
        y = st[name].double() if wide else torch.zeros(b, hk, width, d, dtype=torch.float64, device=DEV)
        for i in range(b):
            if wide:
                for p0 in range(lens[i] // bs * bs, lens[i] + counts[i], bs):
                    lo, hi = max(p0, lens[i]), min(p0 + bs, lens[i] + counts[i])
                    if lo < hi:
                        y[int(st["table"][i, p0 // bs]), lo - p0:hi - p0] = new[name][i, :, lo - lens[i]:hi - lens[i]].transpose(0, 1)
                continue
            had, rows = lens[i] - starts[i], new[name][i, :, :counts[i]].transpose(0, 1)
            held, scale = rows[:0], torch.zeros(hk, dtype=torch.float64, device=DEV)
            if had:
                page = int(st["table"][i, starts[i] // bs])
                held, scale = st[name][page, :had].double(), st[name + "_scales"][page].double()
            if not counts[i]:
                y[i, :, :had] = (held * scale[:, None]).transpose(0, 1)
                continue
            x = torch.cat([held, rows])
            for j in range(0, x.shape[0], bs):
                z = _exact_page(x[j:j + bs], had if j == 0 else 0, scale if j == 0 else 0 * scale, case["pool"])
                y[i, :, j:j + z.shape[0]] = z.transpose(0, 1)
        out[name] = y
    return out


def _exact_attend(st):
    case = st["case"]
    q, hk, d, t, bs = st["q"].double(), case["kv_heads"], case["dim"], case["tokens"], case["page"]
    b, h = q.shape[:2]
    out = torch.zeros_like(q)
    for i, n in enumerate(st["lens"].tolist()):
        pages = st["table"][i, :-(-n // bs)].long()
        held = []
        for name in ("k", "v"):
            x = st[name].view(torch.uint8)[pages].view(st[name].dtype).double()
            held.append((x * st[name + "_scales"][pages].double()[:, None, :, None]).flatten(0, 1)[:n].transpose(0, 1))
        for row in range(t):
            m = n - t + row + 1
            x = torch.einsum("gjd,gnd->gjn", q[i, :, row].view(hk, h // hk, d), held[0][:, :m]) / math.sqrt(d)
            out[i, :, row] = torch.einsum("gjn,gnd->gjd", torch.softmax(x, -1), held[1][:, :m]).reshape(h, d)
    return {"out": out}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "attend":
        return _exact_attend(st)
    w, magnitude = _case_frequencies(case)
    out = {}
    for name in ("q", "k"):
        out[name] = st[name].detach().double()
        for key, sign in ((name, 1.0), ("d" + name, -1.0)):
            if key in st:
                out[key] = _exact_turn(st[key], st["positions"], w.to(DEV), case["interleaved"], sign, magnitude)
    return out


# --------------------------------------------------------------------- work --
def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if kind == "rotary":
        values = b * case["seq"] * (h + hk) * d * (2 if case["train"] else 1)
        return {"bytes": 2 * e * values + 4 * b * case["seq"], "flops": 3 * values * case["rotary"] // d}
    lens, pool = _lengths(case), SIZE[case["pool"]]
    if kind == "append":
        new, bs = _new_lengths(case), case["page"]
        moved = 2 * sum(new) * hk * d * (e + pool) + 2 * b * case["tokens"] * h * d * e
        if pool == 1:  # pages that were open hold tokens that are restated; what is read back counts too
            held = sum(n % bs for n, t in zip(lens, new) if t)
            moved += 2 * held * hk * d + 2 * hk * 4 * sum(-(-(n % bs + t) // bs) for n, t in zip(lens, new))
            width = -(-(case["tokens"] + bs - 1) // bs) * bs
            moved += 2 * hk * d * ((held + sum(new)) * pool + b * width * e)
        return {"bytes": moved, "flops": 3 * (sum(new) * hk + b * case["tokens"] * h) * case["rotary"]}
    lens = [max(n, case["tokens"]) for n in lens]
    t = case["tokens"]
    seen = sum(n * t - t * (t - 1) // 2 for n in lens)
    pages = sum(-(-n // case["page"]) for n in lens)
    return {"bytes": 2 * hk * (sum(lens) * d + 4 * pages) + 4 * pages + 2 * b * h * t * d * e,
            "flops": 4 * d * h * seen}
