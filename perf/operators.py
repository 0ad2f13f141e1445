"""The cases in which the paged-cache operators are measured: page tables built from request
lengths (assignPages), the cache write and read-back (storeKV, loadKV), and attention over the
paged cache for single new tokens and for chunks of them (pagedAttention).

`run` computes each one in a plain form, with elementary torch operations in fp32; with `own` set,
through the calls that a user makes of nim_lowprec_b200.
"""
import math
import random

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # page tables of a decode step: a handful of requests, one token each (latency)
        dict(name="tables decode 7", op="tables", requests=7, new=1, ragged=False, ctx=2000,
             page=16, lens=1),
        # page tables of a large mixed step: prompts of up to 256 tokens beside running requests
        dict(name="tables mixed 1500", op="tables", requests=1500, new=256, ragged=True, ctx=8000,
             page=32, lens=2),
        # one decode step of 61 requests into an int8 cache, from fp32 projections
        dict(name="store int8 61", op="store", tokens=61, kv_heads=8, dim=128, page=16, x="fp32",
             cache="int8"),
        # a prompt of 8191 tokens into an fp16 cache
        dict(name="store fp16 8191", op="store", tokens=8191, kv_heads=8, dim=128, page=16,
             x="fp32", cache="fp16"),
        # a prompt into an int8 cache of a model with one key head per query head
        dict(name="store int8 4096", op="store", tokens=4096, kv_heads=32, dim=128, page=32,
             x="bf16", cache="int8"),
        # one user, one token: 32 heads of their own (Llama-7B's layout), fp32 projections
        dict(name="decode fp32 1", op="attn", requests=1, new=1, ragged=False, ctx=1000, heads=32,
             kv_heads=32, dim=128, page=16, x="fp32", cache="fp16", window=0, sinks=0, lens=3),
        # a served batch at ragged lengths, four query heads to a key head, int8 cache
        dict(name="decode int8 53", op="attn", requests=53, new=1, ragged=True, ctx=16000,
             heads=32, kv_heads=8, dim=128, page=16, x="fp32", cache="int8", window=0, sinks=0,
             lens=4),
        # two long documents, eight query heads to a key head
        dict(name="decode bf16 long", op="attn", requests=2, new=1, ragged=False, ctx=131000,
             heads=64, kv_heads=8, dim=128, page=64, x="bf16", cache="bf16", window=0, sinks=0,
             lens=5),
        # a batch that streams without end: a window and a few first tokens that stay visible
        dict(name="decode window 32", op="attn", requests=32, new=1, ragged=True, ctx=20000,
             heads=64, kv_heads=8, dim=64, page=16, x="bf16", cache="bf16", window=4000, sinks=4,
             lens=6),
        # prompts of fp32 projections over an int8 cache, some with earlier turns
        dict(name="chunk fp32 int8", op="attn", requests=5, new=700, ragged=True, ctx=4000,
             heads=32, kv_heads=32, dim=128, page=16, x="fp32", cache="int8", window=0, sinks=0,
             lens=7),
        # one long prompt's next chunk in 16 bits
        dict(name="chunk bf16 4096", op="attn", requests=1, new=4096, ragged=False, ctx=16384,
             heads=32, kv_heads=8, dim=128, page=32, x="bf16", cache="bf16", window=0, sinks=0,
             lens=8),
        # ragged chunks under a window with sinks, small heads
        dict(name="chunk fp16 window", op="attn", requests=4, new=2500, ragged=True, ctx=6000,
             heads=16, kv_heads=4, dim=64, page=16, x="fp16", cache="fp16", window=1000, sinks=16,
             lens=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "store", "store", "decode", "decode", "decode", "chunk", "chunk",
                       "chunk"])
    lens = rng.randrange(1 << 20)
    page = rng.choice([8, 16, 32, 64, 128])
    if kind == "tables":
        new = rng.choice([1, _log(rng, 2, 256)])
        return dict(op="tables", requests=_log(rng, 1, 1500), new=new, ragged=new > 1,
                    ctx=_log(rng, 16, 8000), page=page, lens=lens)
    if kind == "store":
        return dict(op="store", tokens=_log(rng, 1, 8191), kv_heads=rng.choice([1, 2, 5, 8, 16]),
                    dim=rng.choice([64, 96, 128]), page=page,
                    x=rng.choice(["fp32", "fp16", "bf16"]),
                    cache=rng.choice(["fp16", "bf16", "int8"]))
    x, cache = rng.choice([("fp32", "fp16"), ("fp32", "int8"), ("fp16", "fp16"), ("bf16", "bf16"),
                           ("bf16", "int8")])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 96, 128, 128])
    window = rng.choice([0, 0, _log(rng, 100, 4000)])
    sinks = rng.choice([0, 4, 100]) if window else 0
    if kind == "decode":
        b = _log(rng, 1, 64)
        return dict(op="attn", requests=b, new=1, ragged=b > 1, ctx=_log(rng, 10, 200000 // b),
                    heads=heads, kv_heads=kv, dim=dim, page=page, x=x, cache=cache, window=window,
                    sinks=sinks, lens=lens)
    b = rng.choice([1, 2, 3, 6])
    most = min(4096, 131072 // heads) // b
    return dict(op="attn", requests=b, new=_log(rng, 20, most), ragged=b > 1,
                ctx=_log(rng, 1, 16000 // b), heads=heads, kv_heads=kv, dim=dim, page=page, x=x,
                cache=cache, window=window, sinks=sinks, lens=lens)


def _lengths(case):
    """(context, new) per request: all at the case's figures, or spread below them."""
    r = random.Random(case["lens"])
    b = case["requests"]
    if not case["ragged"]:
        return [case["ctx"]] * b, [case["new"]] * b
    ctx = [0 if r.random() < 0.05 else int(case["ctx"] * r.random()) for _ in range(b)]
    new = [case["new"] if i == 0 else 1 + int((case["new"] - 1) * r.random()) for i in range(b)]
    ctx[0] = case["ctx"]
    return ctx, new


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    ps = case["page"]
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        ctx = [c if i == 0 else max(0, c - seed % 5) for i, c in enumerate(ctx)]
        used = [-(-c // ps) for c in ctx]
        need = [-(-(c + n) // ps) - u for c, n, u in zip(ctx, new, used)]
        width = -(-max(c + n for c, n in zip(*_lengths(case))) // ps) + 3
        pages = sum(used) + sum(need) + 11
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
        mask = torch.arange(width, device="cuda")[None] < _i32(used)[:, None]
        table[mask] = perm[:sum(used)]
        st.update(ctx=_i32(ctx), new=_i32(new), free=perm[sum(used):].clone(), head=_i32([2]),
                  table=table, tokens=sum(new) + 5)
        if own:
            n = st["tokens"]
            st.update(qstart=_i32([0] * (len(ctx) + 1)), seq=_i32([0] * len(ctx)),
                      slots=torch.zeros(n, dtype=torch.int64, device="cuda"),
                      pos=_i32([0] * n), head_out=_i32([0]))
        return st
    hkv, d = case["kv_heads"], case["dim"]
    cdt = torch.int8 if case["cache"] == "int8" else _DT[case["cache"]]
    if case["op"] == "store":
        t = case["tokens"]
        pages = -(-t // ps) + 3
        # projections come as one row per token, k and v side by side; a few channels are large
        ch = 1.0 + 7.0 * (torch.rand(2, hkv, d, generator=g, device="cuda") > 0.97)
        kv = (_randn(g, t, 2, hkv, d) * ch).to(_DT[case["x"]])
        st.update(k=kv[:, 0], v=kv[:, 1],
                  slots=torch.randperm(pages * ps, generator=g, device="cuda")[:t],
                  kpool=torch.zeros(pages, ps, hkv, d, dtype=cdt, device="cuda"),
                  vpool=torch.zeros(pages, ps, hkv, d, dtype=cdt, device="cuda"))
        shape = (t, hkv, d)
        st["outs"] = (torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda"))
        if cdt == torch.int8:
            st["kscale"] = torch.zeros(pages, ps, hkv, device="cuda")
            st["vscale"] = torch.zeros(pages, ps, hkv, device="cuda")
    else:
        ctx, new = _lengths(case)
        seq = [c + n for c, n in zip(ctx, new)]
        used = [-(-s // ps) for s in seq]
        pages, width = sum(used) + 5, max(used) + 2
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(seq), width), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(width, device="cuda")[None] < _i32(used)[:, None]] = perm[:sum(used)]
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        xdt = _DT[case["x"]]
        st.update(q=(1.5 * _randn(g, start[-1], case["heads"], d)).to(xdt), table=table,
                  seq=_i32(seq), qstart=_i32(start), max_new=max(new), max_seq=max(seq))
        if cdt == torch.int8:
            for n in "kv":
                st[n + "pool"] = torch.randint(-127, 128, (pages, ps, hkv, d), generator=g,
                                               device="cuda", dtype=torch.int8)
                st[n + "scale"] = 0.01 + 0.01 * torch.rand(pages, ps, hkv, generator=g,
                                                           device="cuda")
        else:
            for n in "kv":
                st[n + "pool"] = torch.empty(pages, ps, hkv, d, dtype=cdt, device="cuda").normal_(
                    generator=g)
        st["out"] = torch.empty_like(st["q"])
    if own:
        import nim_lowprec_b200 as L
        st["cache"] = L.KVCache(st["kpool"], st["vpool"], st.get("kscale"), st.get("vscale"))
    return st


# ------------------------------------------------------------------ one pass

def run(state):
    return _OPS[state["case"]["op"]][bool(own)](state)


def _tables_own(s):
    import nim_lowprec_b200 as L
    L.assignPages(s["ctx"], s["new"], s["case"]["page"], s["free"], s["head"], s["table"],
                  s["qstart"], s["seq"], s["slots"], s["pos"], s["head_out"])
    return dict(table=s["table"], qstart=s["qstart"], seq=s["seq"], slots=s["slots"], pos=s["pos"],
                head=s["head_out"])


def _tables_plain(s):
    ctx, new, ps, table = s["ctx"].long(), s["new"].long(), s["case"]["page"], s["table"]
    seq = ctx + new
    first, last = (ctx + ps - 1) // ps, (seq + ps - 1) // ps
    need = last - first
    base = torch.cumsum(need, 0) - need + s["head"].long()
    col = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (col >= first[:, None]) & (col < last[:, None])
    take = base[:, None] + col - first[:, None]
    there = fresh & (take < s["free"].numel())
    got = s["free"][torch.where(there, take, torch.zeros_like(take))]
    table = torch.where(there, got, torch.where(fresh, torch.full_like(table, -1), table))
    qend = torch.cumsum(new, 0)
    qstart = torch.cat([torch.zeros_like(qend[:1]), qend])
    t = torch.arange(s["tokens"], device="cuda")
    inside = t < qend[-1]
    req = torch.searchsorted(qend, t, right=True).clamp(max=ctx.numel() - 1)
    pos = torch.where(inside, ctx[req] + t - qstart[req], torch.zeros_like(t))
    page = table[req, pos // ps].long()
    slots = torch.where(inside & (page >= 0), page * ps + pos % ps, torch.full_like(t, -1))
    return dict(table=table, qstart=qstart.int(), seq=seq.int(), slots=slots,
                pos=torch.where(inside, pos, torch.full_like(t, -1)).int(),
                head=torch.minimum(s["head"].long() + need.sum(),
                                   torch.full_like(s["head"].long(), s["free"].numel())).int())


def _store_own(s):
    import nim_lowprec_b200 as L
    L.storeKV(s["cache"], s["k"], s["v"], s["slots"])
    L.loadKV(s["cache"], s["slots"], *s["outs"])
    return s["outs"]


def _write_read(x, slots, pool, scale):
    page, off = slots // pool.shape[1], slots % pool.shape[1]
    x = x.float()
    if scale is None:
        pool[page, off] = x.to(pool.dtype)
        return pool[page, off].float()
    amax = x.abs().amax(-1)
    sc = torch.where(amax == 0, torch.ones_like(amax), amax / torch.full_like(amax, 127.0))
    y = x / sc[..., None]
    pool[page, off] = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-128, 127).to(torch.int8)
    scale[page, off] = sc
    return pool[page, off].float() * scale[page, off][..., None]


def _store_plain(s):
    return (_write_read(s["k"], s["slots"], s["kpool"], s.get("kscale")),
            _write_read(s["v"], s["slots"], s["vpool"], s.get("vscale")))


def _attn_own(s):
    import nim_lowprec_b200 as L
    c = s["case"]
    L.pagedAttention(s["cache"], s["table"], s["qstart"], s["seq"], s["q"], s["out"],
                     window=c["window"], sinks=c["sinks"])
    return s["out"]


def _attn_plain(s):
    c, q, ps = s["case"], s["q"], s["case"]["page"]
    b, hkv, d = s["seq"].numel(), c["kv_heads"], c["dim"]
    grp, nq, nk = c["heads"] // hkv, s["max_new"], s["max_seq"]
    j = torch.arange(nk, device="cuda")
    page = s["table"][:, j // ps].long()
    there = (page >= 0) & (j[None] < s["seq"][:, None])
    page = page.clamp(min=0)
    # keys and values of every request, [requests, kv heads, keys, dim] in fp32
    k, v = s["kpool"][page, j % ps].float(), s["vpool"][page, j % ps].float()
    if c["cache"] == "int8":
        k = k * s["kscale"][page, j % ps][..., None]
        v = v * s["vscale"][page, j % ps][..., None]
    v = torch.where(there[:, :, None, None], v, torch.zeros_like(v))
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    # queries padded to the longest chunk, [requests, kv heads, new x group, dim]
    n = (s["qstart"][1:] - s["qstart"][:-1]).long()
    t = torch.arange(nq, device="cuda")
    row = (s["qstart"][:-1].long()[:, None] + t[None]).clamp(max=q.shape[0] - 1)
    qq = q[row].float().reshape(b, nq, hkv, grp, d).permute(0, 2, 1, 3, 4)
    score = torch.matmul(qq.reshape(b, hkv, nq * grp, d), k.transpose(2, 3)) * (d ** -0.5)
    pos = (s["seq"].long() - n)[:, None] + t[None]
    see = there[:, None, :] & (j[None, None] <= pos[:, :, None])
    if c["window"]:
        see &= (j[None, None] > pos[:, :, None] - c["window"]) | (j[None, None] < c["sinks"])
    score = score.reshape(b, hkv, nq, grp, nk).masked_fill_(~see[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, hkv, nq * grp, nk), v).reshape(b, hkv, nq, grp, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(b, nq, c["heads"], d)
    return o[t[None] < n[:, None]].to(q.dtype)


_OPS = {"tables": (_tables_plain, _tables_own), "store": (_store_plain, _store_own),
        "attn": (_attn_plain, _attn_own)}


# ------------------------------------------------------------------ what a pass cannot do without

_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}


def _seen(case):
    """(keys that some new token sees, query-key pairs), over all requests."""
    keys = pairs = 0
    for c, n in zip(*_lengths(case)):
        w, s = case["window"], case["sinks"]
        if not w:
            keys += c + n
            pairs += n * c + n * (n + 1) // 2
            continue
        lo = max(0, c + 1 - w)  # the first token's window starts here
        keys += c + n - lo + min(s, lo)
        for p in range(c, c + n):
            lo = max(0, p + 1 - w)
            pairs += p + 1 - lo + min(s, lo)
    return keys, pairs


def work(case):
    if case["op"] == "tables":
        ctx, new = _lengths(case)
        b, t, ps = len(ctx), sum(new), case["page"]
        need = sum(-(-(c + n) // ps) + (-c // ps) for c, n in zip(ctx, new))
        # lengths in; free pages read and written to the table; starts, lengths, slots, positions out
        return dict(bytes=8 * b + 8 * need + 8 * b + 4 + 12 * (t + 5) + 8, flops=0)
    rows = _SIZE[case["cache"]] * case["dim"] + (4 if case["cache"] == "int8" else 0)
    if case["op"] == "store":
        n = 2 * case["tokens"] * case["kv_heads"]
        # the rows in, the cache's rows written and read, fp32 rows out; the slots twice
        return dict(bytes=n * (case["dim"] * (_SIZE[case["x"]] + 4) + 2 * rows)
                    + 16 * case["tokens"], flops=n * case["dim"] * 4)
    keys, pairs = _seen(case)
    t = sum(_lengths(case)[1])
    return dict(bytes=2 * keys * case["kv_heads"] * rows
                + 2 * t * case["heads"] * case["dim"] * _SIZE[case["x"]],
                flops=4 * pairs * case["heads"] * case["dim"])


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] == "store":
        return tuple(_exact_round(s[n], case["cache"]) for n in "kv")
    ps, grp = case["page"], case["heads"] // case["kv_heads"]
    ctx, new = _lengths(case)
    outs = []
    for b, (c, n) in enumerate(zip(ctx, new)):
        j = torch.arange(c + n, device="cuda")
        page = s["table"][b, j // ps].long()
        q = s["q"][sum(new[:b]):sum(new[:b]) + n].double() / math.sqrt(case["dim"])
        o = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            k, v = (s[x + "pool"][page, j % ps, h // grp].double() for x in "kv")
            if case["cache"] == "int8":
                k, v = (x * s[m + "scale"][page, j % ps, h // grp].double()[:, None]
                        for x, m in ((k, "k"), (v, "v")))
            for t0 in range(0, n, 1024):
                p = c + torch.arange(t0, min(n, t0 + 1024), device="cuda")[:, None]
                hidden = j[None] > p
                if case["window"]:
                    hidden |= (j[None] <= p - case["window"]) & (j[None] >= case["sinks"])
                a = (q[t0:t0 + 1024, h] @ k.T).masked_fill_(hidden, -math.inf)
                o[t0:t0 + 1024, h] = torch.softmax(a, -1) @ v
        outs.append(o)
    return torch.cat(outs)


def _exact_round(x, cache):
    """What the cache's format can hold of x: fp16 and bf16 by their rounding, int8 by a scale of
    a 127th of the row's largest magnitude."""
    if cache != "int8":
        return x.to(_DT[cache]).double()
    x = x.double()
    scale = x.abs().amax(-1, keepdim=True) / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    y = x / scale
    return torch.sign(y) * torch.floor(y.abs() + 0.5) * scale
