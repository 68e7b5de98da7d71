"""Workloads of the window/sink, draft-tree and cache-page operators.

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
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # Training a long-context model whose layers slide: forward and all three gradients,
        # GQA 32/8, the window of the benchmarked configuration, four sink tokens.
        {"name": "sink_train_bf16_s32768", "kind": "sink_train", "dtype": "bf16", "batch": 1, "heads": 32,
         "kv_heads": 8, "seq": 32768, "dim": 128, "window": 4096, "sinks": 4, "alibi": False},
        # A narrow window over a long sequence (the sinks' own gradient is the long axis here), with ALiBi.
        {"name": "sink_train_bf16_narrow", "kind": "sink_train", "dtype": "bf16", "batch": 2, "heads": 16,
         "kv_heads": 4, "seq": 16384, "dim": 128, "window": 512, "sinks": 16, "alibi": True},
        # Odd length and window, head dim 64, fp16, heads not a power of two.
        {"name": "sink_train_f16_odd", "kind": "sink_train", "dtype": "f16", "batch": 3, "heads": 12,
         "kv_heads": 4, "seq": 1999, "dim": 64, "window": 511, "sinks": 5, "alibi": False},
        # One token per sequence, few sequences: a chat reply streaming out, where latency counts.
        {"name": "window_decode_b1", "kind": "window_decode", "dtype": "bf16", "batch": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "ctx_lo": 20011, "ctx_hi": 20011, "tokens": 1,
         "window": 1024, "sinks": 4},
        # A serving batch of ragged contexts, one token each.
        {"name": "window_decode_b64", "kind": "window_decode", "dtype": "bf16", "batch": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "ctx_lo": 512, "ctx_hi": 32768, "tokens": 1,
         "window": 4096, "sinks": 4},
        # A small tree for one sequence: speculative decoding of a single reply.
        {"name": "tree_b1_t13", "kind": "tree", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "ctx_lo": 2500, "ctx_hi": 2500, "tokens": 13},
        # A batch of ragged contexts, 16 drafted tokens each (64 query rows per kv head).
        {"name": "tree_b64_t16", "kind": "tree", "dtype": "bf16", "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "ctx_lo": 512, "ctx_hi": 32768, "tokens": 16},
        # Wide trees (64 drafted tokens, 512 query rows per kv head), larger pages, fp16.
        {"name": "tree_b8_t64", "kind": "tree", "dtype": "f16", "batch": 8, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "ctx_lo": 1000, "ctx_hi": 16384, "tokens": 64},
        # The accepted path of every sequence goes into its pages.
        {"name": "accept_b64", "kind": "accept", "dtype": "bf16", "batch": 64, "kv_heads": 8, "dim": 128,
         "page": 16, "ctx_lo": 512, "ctx_hi": 4096, "tokens": 64, "depth": 9},
        # Parallel sampling: 48 new rows share the pages of 8 prompts.
        {"name": "fork_b48", "kind": "fork", "dtype": "bf16", "batch": 64, "forks": 48, "kv_heads": 8, "dim": 128,
         "page": 16, "ctx_lo": 500, "ctx_hi": 4000},
        # Half of the sequences end: their pages are freed and the pool is defragmented.
        {"name": "compact_b64", "kind": "compact", "dtype": "bf16", "batch": 64, "ended": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "ctx_lo": 100, "ctx_hi": 4000},
        # Plain page copies (a swap of 2048 pages inside one pool).
        {"name": "copy_2048", "kind": "copy", "dtype": "f16", "blocks": 8192, "copies": 2048, "kv_heads": 8,
         "dim": 128, "page": 16},
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["sink_train", "sink_train", "window_decode", "window_decode", "tree", "tree",
                       "accept", "fork", "compact", "copy"])
    half = rng.choice(["bf16", "bf16", "f16"])
    kvh = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "sink_train":
        dtype = rng.choice([half, half, half, "f32"])
        seq = _logint(rng, 32, 1024 if dtype == "f32" else 16384)
        kvh = min(kvh, 32 // group)
        return {"kind": kind, "dtype": dtype, "batch": rng.choice([1, 2, 3]) if seq < 8192 else 1,
                "heads": kvh * group, "kv_heads": kvh, "seq": seq,
                "dim": dim, "window": _logint(rng, 1, min(seq + 64, 4096)), "sinks": rng.choice([1, 2, 4, 5, 16, 64, 131]),
                "alibi": rng.random() < 0.25}
    hi = _logint(rng, 40, 32768)
    lo = _logint(rng, 1, hi)
    if kind == "window_decode":
        return {"kind": kind, "dtype": half, "batch": _logint(rng, 1, 64), "heads": kvh * group, "kv_heads": kvh,
                "dim": dim, "page": page, "ctx_lo": lo, "ctx_hi": hi, "tokens": rng.choice([1, 1, 1, 2, 3, 7, 20]),
                "window": _logint(rng, 1, 8192), "sinks": rng.choice([0, 1, 4, 4, 17, 128])}
    if kind == "tree":
        hi = min(hi, 16384)
        return {"kind": kind, "dtype": half, "batch": _logint(rng, 1, 32), "heads": kvh * group, "kv_heads": kvh,
                "dim": dim, "page": page, "ctx_lo": min(lo, hi), "ctx_hi": hi, "tokens": _logint(rng, 1, 130)}
    if kind == "accept":
        t = _logint(rng, 1, 96)
        return {"kind": kind, "dtype": half, "batch": _logint(rng, 1, 200), "kv_heads": kvh, "dim": dim, "page": page,
                "ctx_lo": min(lo, 2000), "ctx_hi": min(hi, 2000), "tokens": t, "depth": rng.randint(1, t)}
    if kind == "fork":
        b = _logint(rng, 2, 96)
        return {"kind": kind, "dtype": half, "batch": b, "forks": rng.randint(1, b - 1), "kv_heads": kvh, "dim": dim,
                "page": page, "ctx_lo": min(lo, 3000), "ctx_hi": min(hi, 3000)}
    if kind == "compact":
        b = _logint(rng, 2, 64)
        return {"kind": kind, "dtype": half, "batch": b, "ended": rng.randint(1, b), "kv_heads": kvh, "dim": dim,
                "page": page, "ctx_lo": min(lo, 3000), "ctx_hi": min(hi, 3000)}
    blocks = _logint(rng, 4, 6000)
    return {"kind": "copy", "dtype": half, "blocks": blocks, "copies": rng.randint(1, blocks // 2), "kv_heads": kvh,
            "dim": dim, "page": rng.choice([16, 32])}


# ----------------------------------------------------------------- prepare --
def _gens(seed):
    c = torch.Generator()
    c.manual_seed(seed)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return c, g


def _randn(g, shape, dt):
    # half types are drawn in their own type; the pools are gigabytes
    return torch.randn(shape, generator=g, device=DEV, dtype=dt)


def _lengths(case, c):
    return [int(x) for x in torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (case["batch"],), generator=c)]


def _paged(case, lens, room, c, g, extra=0):
    """Pools, table, lengths: every sequence holds ceil((len + room) / page) pages at random places.

    The pools that a call writes hold the longest sequences of the case; the pools that it only reads
    hold what there is."""
    bs, dt = case["page"], DTYPES[case["dtype"]]
    need = [-(-(n + room) // bs) for n in lens]
    most = -(-(case["ctx_hi"] + room) // bs)
    reads = case["kind"] in ("window_decode", "tree")
    nb = (sum(need) if reads else most * len(lens)) + 2 + extra
    perm = torch.randperm(nb, generator=c).to(torch.int32)
    table = torch.full((len(lens), max(most, 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    shape = (nb, bs, case["kv_heads"], case["dim"])
    return {"k": _randn(g, shape, dt), "v": _randn(g, shape, dt), "table": table.to(DEV),
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "spare": perm[at:].to(DEV), "host_lens": lens,
            "pages": need}


def _tree(batch, tokens, c):
    """Random trees: parents come before their children, -1 hangs a token on the context."""
    par = torch.full((batch, tokens), -1, dtype=torch.int32)
    for t in range(1, tokens):
        back = torch.randint(0, min(t, 6) + 1, (batch,), generator=c)  # one of the last tokens, or a new root
        par[:, t] = torch.where(back == 0, torch.full_like(back, -1 if t < 4 else t - 1), t - back).to(torch.int32)
    return par


def prepare(case, seed):
    c, g = _gens(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "sink_train":
        dt = DTYPES[case["dtype"]]
        b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["dim"]
        st["q"] = _randn(g, (b, h, s, d), dt).requires_grad_(True)
        st["k"] = _randn(g, (b, hk, s, d), dt).requires_grad_(True)
        st["v"] = _randn(g, (b, hk, s, d), dt).requires_grad_(True)
        st["do"] = _randn(g, (b, h, s, d), dt)
        if own:
            import attnax_b200 as ax

            mod = ax.sink_window_mod(case["window"], case["sinks"])
            st["mod"] = ax.compose_score_mods(mod, ax.alibi_mod(h)) if case["alibi"] else mod
        return st
    if kind == "copy":
        shape = (case["blocks"], case["page"], case["kv_heads"], case["dim"])
        dt = DTYPES[case["dtype"]]
        perm = torch.randperm(case["blocks"], generator=c).to(torch.int32).to(DEV)
        n = case["copies"]
        st.update(k=_randn(g, shape, dt), v=_randn(g, shape, dt), src=perm[:n].contiguous(),
                  dst=perm[n:2 * n].contiguous(), table=torch.full((1, 1), -1, dtype=torch.int32, device=DEV),
                  lens=torch.zeros(1, dtype=torch.int32, device=DEV))
    else:
        lens = _lengths(case, c)
        b = case["batch"]
        if kind == "window_decode":
            lens = [max(n, case["tokens"]) for n in lens]
            st.update(_paged(case, lens, 0, c, g))
            st["q"] = _randn(g, (b, case["heads"], case["tokens"], case["dim"]), DTYPES[case["dtype"]])
        elif kind == "tree":
            t, d, dt = case["tokens"], case["dim"], DTYPES[case["dtype"]]
            st.update(_paged(case, lens, 0, c, g))
            st["q"] = _randn(g, (b, case["heads"], t, d), dt)
            # the projections' layout: (batch, tokens, heads, dim), seen as (batch, heads, tokens, dim)
            st["dk"] = _randn(g, (b, t, case["kv_heads"], d), dt).transpose(1, 2)
            st["dv"] = _randn(g, (b, t, case["kv_heads"], d), dt).transpose(1, 2)
            st["parents"] = _tree(b, t, c).to(DEV)
            # a padded batch: trees of different sizes
            st["host_tree"] = [int(x) for x in torch.randint((t + 1) // 2, t + 1, (b,), generator=c)]
            st["tree_lens"] = torch.tensor(st["host_tree"], dtype=torch.int32, device=DEV)
        elif kind == "accept":
            t, d, dt, a = case["tokens"], case["dim"], DTYPES[case["dtype"]], case["depth"]
            st.update(_paged(case, lens, a, c, g))
            st["dk"] = _randn(g, (b, t, case["kv_heads"], d), dt).transpose(1, 2)
            st["dv"] = _randn(g, (b, t, case["kv_heads"], d), dt).transpose(1, 2)
            acc = torch.stack([torch.sort(torch.randperm(t, generator=c)[:a])[0] for _ in range(b)])
            st["host_n"] = [int(x) for x in torch.randint(0, a + 1, (b,), generator=c)]
            st["accepted"] = acc.to(torch.int32).to(DEV)
            st["accepted_lens"] = torch.tensor(st["host_n"], dtype=torch.int32, device=DEV)
        elif kind == "fork":
            f = case["forks"]
            for i in range(b - f, b):
                lens[i] = 0  # the rows that the forks take
            st.update(_paged(case, lens, 0, c, g, extra=f))
            src = torch.randint(0, max(1, min(8, b - f)), (f,), generator=c)
            st["host_src"], st["host_dst"] = src.tolist(), list(range(b - f, b))
            st["src"] = src.to(torch.int32).to(DEV)
            st["dst"] = torch.arange(b - f, b, dtype=torch.int32, device=DEV)
        elif kind == "compact":
            st.update(_paged(case, lens, 0, c, g, extra=7))
            rows = torch.randperm(b, generator=c)[:case["ended"]]
            st["host_ended"] = rows.tolist()
            st["ended"] = rows.to(torch.int32).to(DEV)
        st["max_ctx"] = max(lens) if lens else 0
    if own:
        import attnax_b200 as ax

        st["cache"] = ax.PagedKVCache(st["k"], st["v"], st["table"], st["lens"])
    return st


# --------------------------------------------------------------- plain forms --
def _slopes(n):
    def pow2(m):
        start = 2.0 ** (-(2.0 ** -(math.log2(m) - 3)))
        return [start ** (i + 1) for i in range(m)]

    if n & (n - 1) == 0:
        return pow2(n)
    m = 2 ** int(math.log2(n))
    return pow2(m) + pow2(2 * m)[0::2][:n - m]


def _plain_sink_train(st):
    case = st["case"]
    dt = st["q"].dtype
    q, k, v, do = (st[x].detach().float() for x in ("q", "k", "v", "do"))
    b, h, s, d = q.shape
    hk = k.shape[1]
    grp = h // hk
    w, ns = case["window"], case["sinks"]
    scale = 1.0 / math.sqrt(d)
    n = b * hk
    q = q.reshape(n, grp, s, d)
    do = do.reshape(n, grp, s, d)
    k, v = k.reshape(n, s, d), v.reshape(n, s, d)
    out, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    slopes = None
    if case["alibi"]:
        slopes = torch.tensor(_slopes(h), device=DEV).view(hk, grp).repeat(b, 1)  # (n, grp)
    block = 1024
    for i0 in range(0, s, block):
        i1 = min(s, i0 + block)
        lo = max(0, i0 - w + 1)
        sk = min(ns, lo)
        cols = torch.cat([torch.arange(sk, device=DEV), torch.arange(lo, i1, device=DEV)])
        rows = torch.arange(i0, i1, device=DEV)
        dist = rows[:, None] - cols[None, :]
        keep = (dist >= 0) & ((dist < w) | (cols < ns)[None, :])
        kb, vb = torch.cat([k[:, :sk], k[:, lo:i1]], 1), torch.cat([v[:, :sk], v[:, lo:i1]], 1)
        qb, gb = q[:, :, i0:i1].reshape(n, -1, d), do[:, :, i0:i1].reshape(n, -1, d)
        x = (qb @ kb.transpose(1, 2)).view(n, grp, i1 - i0, -1) * scale
        if slopes is not None:
            x = x - slopes[:, :, None, None] * dist.abs()
        x = x.masked_fill(~keep, float("-inf"))
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).reshape(n, grp * (i1 - i0), -1)
        ob = p @ vb
        dp = gb @ vb.transpose(1, 2)
        ds = p * (dp - (gb * ob).sum(-1, keepdim=True)) * scale
        out[:, :, i0:i1] = ob.view(n, grp, i1 - i0, d)
        dq[:, :, i0:i1] = (ds @ kb).view(n, grp, i1 - i0, d)
        dkb, dvb = ds.transpose(1, 2) @ qb, p.transpose(1, 2) @ gb
        dk[:, :sk] += dkb[:, :sk]
        dk[:, lo:i1] += dkb[:, sk:]
        dv[:, :sk] += dvb[:, :sk]
        dv[:, lo:i1] += dvb[:, sk:]
    return {"out": out.view(b, h, s, d).to(dt), "dq": dq.view(b, h, s, d).to(dt),
            "dk": dk.view(b, hk, s, d).to(dt), "dv": dv.view(b, hk, s, d).to(dt)}


def _rows_of(st, i, toks):
    """Pool rows of tokens ``toks`` of sequence i."""
    bs = st["case"]["page"]
    return st["table"][i].long()[toks // bs] * bs + toks % bs


def _softmax_pv(x, keep, v):
    x = x.masked_fill(~keep, float("-inf"))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    return (p / p.sum(-1, keepdim=True)) @ v


def _plain_window_decode(st):
    case = st["case"]
    q = st["q"]
    b, h, t, d = q.shape
    hk = case["kv_heads"]
    out = torch.empty_like(q)
    kf, vf = st["k"].view(-1, hk, d), st["v"].view(-1, hk, d)
    for i, n in enumerate(st["host_lens"]):
        lo = max(0, n - t - case["window"] + 1)
        sk = min(case["sinks"], lo)
        toks = torch.cat([torch.arange(sk, device=DEV), torch.arange(lo, n, device=DEV)])
        rows = _rows_of(st, i, toks)
        k, v = kf[rows].float().transpose(0, 1), vf[rows].float().transpose(0, 1)  # (hk, n, d)
        qi = q[i].float().view(hk, (h // hk) * t, d)
        pos = torch.arange(n - t, n, device=DEV).repeat(h // hk)
        dist = pos[:, None] - toks[None, :]
        keep = (dist >= 0) & ((dist < case["window"]) | (toks < case["sinks"])[None, :])
        o = _softmax_pv(qi @ k.transpose(1, 2) / math.sqrt(d), keep, v)
        out[i] = o.view(h, t, d).to(q.dtype)
    return out


def _plain_tree(st):
    case = st["case"]
    q = st["q"]
    b, h, t, d = q.shape
    hk = case["kv_heads"]
    grp = h // hk
    out = torch.zeros_like(q)
    # ancestors-or-self, by following the parents level by level
    idx = torch.arange(t, device=DEV).expand(b, t)
    anc = torch.zeros(b, t, t, dtype=torch.bool, device=DEV)
    cur, alive = idx.clone(), torch.ones(b, t, dtype=torch.bool, device=DEV)
    par = st["parents"].long()
    for _ in range(t):
        anc |= (cur.clamp(min=0)[:, :, None] == idx[:, None, :]) & alive[:, :, None]
        cur = torch.where(alive, torch.gather(par, 1, cur.clamp(min=0)), cur)
        alive = alive & (cur >= 0)
    kf, vf = st["k"].view(-1, hk, d), st["v"].view(-1, hk, d)
    for i, n in enumerate(st["host_lens"]):
        m = st["host_tree"][i]
        rows = _rows_of(st, i, torch.arange(n, device=DEV))
        k = torch.cat([kf[rows].float().transpose(0, 1), st["dk"][i, :, :m].float()], 1)
        v = torch.cat([vf[rows].float().transpose(0, 1), st["dv"][i, :, :m].float()], 1)
        qi = q[i, :, :m].float().reshape(hk, grp * m, d)
        keep = torch.cat([torch.ones(m, n, dtype=torch.bool, device=DEV), anc[i, :m, :m]], 1).repeat(grp, 1)
        o = _softmax_pv(qi @ k.transpose(1, 2) / math.sqrt(d), keep, v)
        out[i, :, :m] = o.view(h, m, d).to(q.dtype)
    return out


def _plain_accept(st):
    case = st["case"]
    b = case["batch"]
    bs, hk, d = case["page"], case["kv_heads"], case["dim"]
    a = torch.arange(case["depth"], device=DEV)
    n = st["accepted_lens"].long()
    pos = st["lens"].long()[:, None] + a
    ok = a[None, :] < n[:, None]
    page = torch.gather(st["table"].long(), 1, (pos // bs).clamp(max=st["table"].shape[1] - 1))
    dst = (page * bs + pos % bs)[ok]
    seq = torch.arange(b, device=DEV)[:, None].expand_as(pos)[ok]
    tok = st["accepted"].long()[ok]
    st["k"].view(-1, hk, d)[dst] = st["dk"][seq, :, tok]
    st["v"].view(-1, hk, d)[dst] = st["dv"][seq, :, tok]
    return {"k": st["k"], "v": st["v"], "lens": st["lens"] + st["accepted_lens"]}


def _plain_fork(st):
    bs = st["case"]["page"]
    src, dst = st["src"].long(), st["dst"].long()
    table, lens = st["table"].clone(), st["lens"].clone()
    n = st["lens"].long()[src]
    tail = n % bs != 0
    used = tail.long().cumsum(0)
    rows = st["table"][src]
    fresh = st["spare"][(used - 1).clamp(min=0)]
    col = (n // bs).clamp(max=table.shape[1] - 1)
    old = torch.gather(rows, 1, col[:, None])[:, 0]
    rows.scatter_(1, col[:, None], torch.where(tail, fresh, old)[:, None])
    keep = torch.arange(table.shape[1], device=DEV)[None, :] < ((n + bs - 1) // bs)[:, None]
    table[dst] = torch.where(keep, rows, torch.full_like(rows, -1))
    lens[dst] = st["lens"][src]
    s, f = old[tail].long(), fresh[tail].long()
    st["k"][f] = st["k"][s]
    st["v"][f] = st["v"][s]
    return {"k": st["k"], "v": st["v"], "table": table, "lens": lens, "used": used[-1].to(torch.int32)}


def _plain_compact(st):
    nb = st["k"].shape[0]
    table, lens = st["table"].clone(), st["lens"].clone()
    ended = st["ended"].long()

    def marks(rows):
        m = torch.zeros(nb + 1, dtype=torch.bool, device=DEV)
        e = rows.long().flatten()
        m[torch.where(e < 0, torch.full_like(e, nb), e)] = True
        return m[:nb]

    gone = marks(table[ended])
    table[ended] = -1
    lens[ended] = 0
    live = marks(table)
    freed = torch.full((nb,), -1, dtype=torch.int32, device=DEV)
    ids = torch.nonzero(gone & ~live)[:, 0].to(torch.int32)
    freed[:ids.numel()] = ids
    count = torch.tensor(ids.numel(), dtype=torch.int32, device=DEV)
    n_live = int(live.sum())
    holes = torch.nonzero(~live[:n_live])[:, 0]
    movers = torch.nonzero(live[n_live:])[:, 0] + n_live
    remap = torch.arange(nb, device=DEV, dtype=torch.int32)
    remap[movers] = holes.to(torch.int32)
    st["k"][holes] = st["k"][movers]
    st["v"][holes] = st["v"][movers]
    new = torch.where(table < 0, table, remap[table.clamp(min=0).long()])
    return {"k": st["k"], "v": st["v"], "table": new, "lens": lens, "freed": freed, "num_freed": count,
            "num_live": torch.tensor(n_live, dtype=torch.int32, device=DEV)}


def _plain_copy(st):
    s, d = st["src"].long(), st["dst"].long()
    st["k"][d] = st["k"][s]
    st["v"][d] = st["v"][s]
    return {"k": st["k"], "v": st["v"]}


# --------------------------------------------------------------------- own --
def _own(st):
    import attnax_b200 as ax

    case = st["case"]
    kind = case["kind"]
    if kind == "sink_train":
        out = ax.flash_attention(st["q"], st["k"], st["v"], score_mod=st["mod"])
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    cache = st["cache"]
    if kind == "window_decode":
        return ax.paged_window_attention(st["q"], cache, window_size=case["window"], num_sinks=case["sinks"],
                                         max_context=st["max_ctx"])
    if kind == "tree":
        return ax.paged_tree_attention(st["q"], st["dk"], st["dv"], cache, st["parents"],
                                       tree_lengths=st["tree_lens"], max_context=st["max_ctx"])
    if kind == "accept":
        new = ax.append_accepted(cache, st["dk"], st["dv"], st["accepted"], st["accepted_lens"], check=False)
        return {"k": new.key_pool, "v": new.value_pool, "lens": new.seq_lengths}
    if kind == "fork":
        new, used = ax.fork_sequences(cache, st["src"], st["dst"], st["spare"])
        return {"k": new.key_pool, "v": new.value_pool, "table": new.block_table, "lens": new.seq_lengths,
                "used": used}
    if kind == "compact":
        new, freed, count = ax.free_sequences(cache, st["ended"])
        new, live = ax.compact_blocks(new)
        return {"k": new.key_pool, "v": new.value_pool, "table": new.block_table, "lens": new.seq_lengths,
                "freed": freed, "num_freed": count, "num_live": live}
    new = ax.copy_blocks(cache, st["src"], st["dst"])
    return {"k": new.key_pool, "v": new.value_pool}


_PLAIN = {"sink_train": _plain_sink_train, "window_decode": _plain_window_decode, "tree": _plain_tree,
          "accept": _plain_accept, "fork": _plain_fork, "compact": _plain_compact, "copy": _plain_copy}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work --
def _visible(n, window, sinks):
    """Kept (q, kv) pairs of a causal window with sinks over n positions."""
    w = min(window, n)
    pairs = w * (w + 1) // 2 + (n - w) * w
    for c in range(min(sinks, n)):
        pairs += max(0, n - c - w)
    return pairs


def work(case):
    kind = case["kind"]
    e = SIZE[case["dtype"]]
    if kind == "sink_train":
        b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["seq"], case["dim"]
        pairs = _visible(s, case["window"], case["sinks"])
        # reads q, do, k, v; writes out, dq, dk, dv
        return {"bytes": e * b * s * d * (4 * h + 4 * hk), "flops": 14 * d * h * b * pairs}
    if kind == "copy":
        return {"bytes": 4 * case["copies"] * case["page"] * case["kv_heads"] * case["dim"] * e, "flops": 0}
    mean = (case["ctx_lo"] + case["ctx_hi"]) / 2
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    if kind == "window_decode":
        t, h = case["tokens"], case["heads"]
        span = case["ctx_hi"] - case["ctx_lo"] + 1
        cap = case["window"] + t - 1 + case["sinks"]
        step = max(1, span // 997)
        ctx = [min(max(n, t), cap) for n in range(case["ctx_lo"], case["ctx_hi"] + 1, step)]
        keys = sum(ctx) / len(ctx)
        return {"bytes": int(e * b * (2 * keys * hk * d + 2 * h * t * d) + 4 * b * keys / case["page"]),
                "flops": int(4 * d * h * t * b * keys)}
    if kind == "tree":
        t, h = 0.75 * case["tokens"], case["heads"]
        return {"bytes": int(e * b * (2 * (mean + t) * hk * d + 2 * h * t * d) + 4 * b * mean / case["page"]),
                "flops": int(4 * d * h * t * b * (mean + t / 4))}
    row = hk * d * e
    if kind == "accept":
        return {"bytes": int(4 * b * case["depth"] / 2 * row), "flops": 0}
    pages = b * (mean / case["page"] + 1)
    if kind == "fork":
        return {"bytes": int(4 * case["forks"] * case["page"] * row + 8 * pages), "flops": 0}
    live = pages * (1 - case["ended"] / b)
    moved = live * (1 - live / (pages + 9))  # live pages behind the first `live` ones, at random places
    return {"bytes": int(4 * moved * case["page"] * row + 16 * pages), "flops": 0}


# ------------------------------------------------------------------- exact --
def _exact_train(st):
    """Whole score rows in 64 bits with the mask written out over all keys."""
    case = st["case"]
    q, k, v, do = (st[x].detach().double() for x in ("q", "k", "v", "do"))
    b, h, s, d = q.shape
    grp = h // k.shape[1]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    kv = torch.arange(s, device=DEV)
    slopes = _slopes(h)
    step = max(1, min(s, (1 << 27) // s))
    for i0 in range(0, s, step):
        r = torch.arange(i0, min(s, i0 + step), device=DEV)
        drop = (kv[None] > r[:, None]) | ((r[:, None] - kv[None] >= case["window"]) & (kv[None] >= case["sinks"]))
        for bi in range(b):
            for hi in range(h):
                kk, vv = k[bi, hi // grp], v[bi, hi // grp]
                x = torch.mm(q[bi, hi, r], kk.t()).div_(math.sqrt(d))
                if case["alibi"]:
                    x -= slopes[hi] * (r[:, None] - kv[None]).abs()
                p = torch.softmax(x.masked_fill_(drop, -math.inf), -1)
                del x
                g = do[bi, hi, r]
                o = torch.mm(p, vv)
                out[bi, hi, r] = o
                dv[bi, hi // grp] += torch.mm(p.t(), g)
                ds = torch.mm(g, vv.t()).sub_((g * o).sum(1)[:, None]).mul_(p)
                dq[bi, hi, r] = torch.mm(ds, kk) / math.sqrt(d)
                dk[bi, hi // grp] += torch.mm(ds.t(), q[bi, hi, r]) / math.sqrt(d)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _history(st, i, name):
    """All cached tokens of sequence i, page by page: (tokens, heads, dim) in 64 bits."""
    n, bs = st["host_lens"][i], st["case"]["page"]
    pages = st["table"][i, :-(-n // bs)].long()
    return st[name].index_select(0, pages).double().flatten(0, 1)[:n]


def _exact_decode(st):
    case = st["case"]
    q = st["q"].double()
    b, h, t, d = q.shape
    grp = h // case["kv_heads"]
    out = torch.zeros_like(q)
    for i in range(b):
        n = st["host_lens"][i]
        k, v = _history(st, i, "k"), _history(st, i, "v")
        if case["kind"] == "tree":
            m = st["host_tree"][i]
            par = st["parents"][i].tolist()
            see = torch.zeros(m, n + m, dtype=torch.bool)
            see[:, :n] = True
            for r in range(m):
                if par[r] >= 0:
                    see[r, n:] = see[par[r], n:]
                see[r, n + r] = True
            k = torch.cat([k, st["dk"][i, :, :m].double().permute(1, 0, 2)])
            v = torch.cat([v, st["dv"][i, :, :m].double().permute(1, 0, 2)])
        else:
            m = t
            p = torch.arange(n)
            see = torch.zeros(m, n, dtype=torch.bool)
            for r in range(m):
                at = n - t + r
                see[r] = (p <= at) & ((p > at - case["window"]) | (p < case["sinks"]))
        see = see.to(DEV)
        for j in range(h):
            x = torch.einsum("td,nd->tn", q[i, j, :m], k[:, j // grp]) / math.sqrt(d)
            out[i, j, :m] = torch.softmax(x.masked_fill(~see, -math.inf), 1) @ v[:, j // grp]
    return out


def _exact_pages(st):
    """The page operators on host tables, one entry after the other."""
    case = st["case"]
    kind, bs = case["kind"], case.get("page")
    k, v = st["k"].double(), st["v"].double()
    table, lens = st["table"].tolist(), st["lens"].tolist()
    res = {}
    moves = []
    if kind == "copy":
        moves = list(zip(st["src"].tolist(), st["dst"].tolist()))
    elif kind == "accept":
        acc = st["accepted"].tolist()
        for i, n in enumerate(st["host_n"]):
            for j in range(n):
                page, row = table[i][(lens[i] + j) // bs], (lens[i] + j) % bs
                k[page, row] = st["dk"][i, :, acc[i][j]].double()
                v[page, row] = st["dv"][i, :, acc[i][j]].double()
        return {"k": k, "v": v, "lens": torch.tensor([a + n for a, n in zip(lens, st["host_n"])], dtype=torch.int32)}
    elif kind == "fork":
        spare, used = st["spare"].tolist(), 0
        new, newlen = [list(r) for r in table], list(lens)
        for s, t in zip(st["host_src"], st["host_dst"]):
            n = -(-lens[s] // bs)
            new[t] = table[s][:n] + [-1] * (len(table[s]) - n)
            newlen[t] = lens[s]
            if lens[s] % bs:
                moves.append((table[s][n - 1], spare[used]))
                new[t][n - 1] = spare[used]
                used += 1
        res = {"table": new, "lens": newlen, "used": used}
    elif kind == "compact":
        nb = k.shape[0]
        gone = {p for i in st["host_ended"] for p in table[i] if p >= 0}
        for i in st["host_ended"]:
            table[i], lens[i] = [-1] * len(table[i]), 0
        live = {p for r in table for p in r if p >= 0}
        freed = sorted(gone - live)
        holes = [p for p in range(len(live)) if p not in live]
        moves = list(zip(sorted(p for p in live if p >= len(live)), holes))
        to = dict(moves)
        res = {"table": [[to.get(p, p) for p in r] for r in table], "lens": lens,
               "freed": freed + [-1] * (nb - len(freed)), "num_freed": len(freed), "num_live": len(live)}
    if moves:
        s, d = (torch.tensor(x, device=DEV) for x in zip(*moves))
        k[d], v[d] = k[s], v[s]
    return {"k": k, "v": v, **{n: torch.tensor(x, dtype=torch.int32) for n, x in res.items()}}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "sink_train":
        return _exact_train(st)
    if case["kind"] in ("window_decode", "tree"):
        return _exact_decode(st)
    return _exact_pages(st)
