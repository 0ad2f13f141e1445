"""Plain 64-bit forms of the paged cache's operators, and inputs for their tests."""
import math

import numpy as np
import torch

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
#: half a unit in the last place, relative: what one rounding to the type costs
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def assign_pages(ctx, new, ps, free, head, table, tokens):
    """numpy, request by request; `table` is changed in place."""
    qstart, seq, slots, pos = [0], [], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        first = min(-(-c // ps), table.shape[1])
        last = min(-(-(c + n) // ps), table.shape[1])
        for i in range(first, last):
            table[b, i] = free[head] if head < len(free) else -1
            head += 1
        for p in range(c, c + n):
            at = p // ps
            page = table[b, at] if at < table.shape[1] else -1
            slots.append(page * ps + p % ps if page >= 0 else -1)
            pos.append(p)
        qstart.append(qstart[-1] + n)
        seq.append(c + n)
    pad = max(0, tokens - len(slots))
    slots, pos = (slots + [-1] * pad)[:tokens], (pos + [-1] * pad)[:tokens]
    return dict(table=table, qstart=qstart, seq=seq, slots=slots, pos=pos,
                head=max(min(head, len(free)), 0))


def quantize_rows(x):
    """calibrateSymmetric(groupSize = row, qmax 127) and quantizeBatch in numpy fp32."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1)
    s = np.where(amax == 0, np.float32(1), amax / np.float32(127)).astype(np.float32)
    y = (x / s[..., None]).astype(np.float32)
    q = np.clip(np.sign(y) * np.floor(np.abs(y) + np.float32(0.5)), -128, 127)
    return q.astype(np.int8), s


def dequant_cache(cache):
    """(k, v) of a cache in 64 bits, [pages, pageSize, kvHeads, headDim]."""
    out = []
    for t, s in ((cache.k, cache.kScales), (cache.v, cache.vScales)):
        t = t.double()
        out.append(t if s is None else t * s.double()[..., None])
    return out


def attention(cache, table, qstart, seqlens, q, scale, window=0, sinks=0):
    """(out, lse, a, s) in 64 bits: a = sum p |v| / sum p and s = the row's largest
    sum |scale q k|, which bound the error of a computation in fewer bits."""
    kd, vd = dequant_cache(cache)
    pages, ps, hkv, d = kd.shape
    t_all, hq, _ = q.shape
    grp = hq // hkv
    out = torch.zeros(t_all, hq, d, dtype=torch.float64, device=q.device)
    amp = torch.zeros_like(out)
    lse = torch.full((t_all, hq), -math.inf, dtype=torch.float64, device=q.device)
    big = torch.zeros(t_all, hq, dtype=torch.float64, device=q.device)
    starts, lens = qstart.tolist(), seqlens.tolist()
    for b, seq in enumerate(lens):
        t0, t1 = starts[b], starts[b + 1]
        n = t1 - t0
        keys = min(seq, table.shape[1] * ps)
        if n == 0 or keys <= 0:
            continue
        j = torch.arange(keys, device=q.device)
        page = table[b, j // ps].long()
        there = (page >= 0) & (page < pages)
        page = torch.where(there, page, torch.zeros_like(page))
        k, v = kd[page, j % ps], vd[page, j % ps]
        p = (seq - n + torch.arange(n, device=q.device))[:, None]
        see = there[None] & (j[None] <= p)
        if window:
            see &= (j[None] > p - window) | (j[None] < sinks)
        some = see.any(0)  # keys that nobody sees may hold anything
        k, v = (torch.where(some[:, None, None], x, torch.zeros_like(x)) for x in (k, v))
        for h in range(hq):
            qq, kk, vv = q[t0:t1, h].double(), k[:, h // grp], v[:, h // grp]
            sc = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            top = sc.amax(1, keepdim=True)
            w = torch.exp(sc - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
            w = torch.where(see, w, torch.zeros_like(w))
            tot = w.sum(1, keepdim=True)
            if torch.isfinite(vv).all():
                o, av = w @ vv, w @ vv.abs()
            else:  # a masked key's value must not meet its weight of zero
                o = torch.stack([(w[i][see[i], None] * vv[see[i]]).sum(0) for i in range(n)])
                av = torch.stack([(w[i][see[i], None] * vv[see[i]].abs()).sum(0)
                                  for i in range(n)])
            safe = torch.where(tot > 0, tot, torch.ones_like(tot))
            out[t0:t1, h], amp[t0:t1, h] = o / safe, av / safe
            lse[t0:t1, h] = (torch.log(tot) + torch.where(torch.isfinite(top), top,
                                                          torch.full_like(top, -math.inf)))[:, 0]
            big[t0:t1, h] = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~see, 0).amax(1)
    return out, lse, amp, big


def tolerance(o, amp, big, dtype):
    """Derived for products of 22-bit or exact operands and fp32 sums.

    A score's error is at most 2^-20 of its sum of magnitudes s (the split's 2^-22, and 16 sums
    of 16 products at 2^-24 each), so a weight's relative error is 2^-20 (s + 1) with the
    exponential's own, in the numerator and in the denominator: 2^-19 (s + 1) a.  A 16-bit
    output rounds once (half an ulp of o); where 16-bit queries run on the chunk kernel each
    weight rounds once to the same type (half an ulp of a)."""
    t = 2.0 ** -19 * (big[..., None] + 1) * amp
    if dtype != torch.float32:
        t = t + HALF_ULP[dtype] * (o.abs() + amp) * 1.001 + 2.0 ** -24
    return t + 1e-30


def lse_tolerance(lse, big):
    return 2.0 ** -19 * (big + 1) + 2.0 ** -22 * torch.where(torch.isfinite(lse), lse.abs(),
                                                             torch.zeros_like(lse))


def make(seed, lens, heads, kv_heads, dim, ps, x="fp32", cache="fp16", tail=None, spare=3,
         heads_first=False, q_scale=1.5):
    """A cache, its tables and queries for requests of (context, new) tokens.  `tail` fills the
    cache's places that belong to no key."""
    import nim_lowprec_b200 as L
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")
    seq = [c + n for c, n in lens]
    used = [max(0, -(-s // ps)) for s in seq]
    pages, width = sum(used) + spare, max(used + [1]) + 1
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(seq), width), -1, dtype=torch.int32, device="cuda")
    at, mine = 0, torch.zeros(pages, ps, dtype=torch.bool, device="cuda")
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        j = torch.arange(max(seq[b], 0), device="cuda")
        mine[perm[at:at + u].long()[j // ps], j % ps] = True
        at += u
    shape = (pages, kv_heads, ps, dim) if heads_first else (pages, ps, kv_heads, dim)

    def view(t):
        return t.transpose(1, 2) if heads_first else t
    if cache == "int8":
        k, v = (view(torch.randint(-128, 128, shape, generator=g, device="cuda",
                                   dtype=torch.int8)) for _ in range(2))
        # scales over many octaves: a few values are far larger than the rest
        ks = 0.02 * torch.exp2(randn(pages, ps, kv_heads) * 0.5)
        vs = torch.exp2(3 * randn(pages, ps, kv_heads))
        if tail is not None:
            ks[~mine], vs[~mine] = tail, tail
        c = L.KVCache(k, v, ks, vs)
    else:
        k, v = (view(randn(*shape).to(DT[cache])) for _ in range(2))
        if tail is not None:
            k[~mine], v[~mine] = tail, tail
        c = L.KVCache(k, v)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    q = (q_scale * randn(starts[-1], heads, dim)).to(DT[x])
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(cache=c, table=table, qstart=torch.tensor(starts, **i32),
                seq=torch.tensor(seq, **i32), q=q)


def check(m, scale=None, window=0, sinks=0, out=None, lse=True, workspace=None):
    """Run pagedAttention on make()'s inputs and hold it to the 64-bit form; returns out."""
    import nim_lowprec_b200 as L
    q = m["q"]
    out = torch.full_like(q, math.nan) if out is None else out
    ls = torch.full(q.shape[:2], math.nan, dtype=torch.float32, device="cuda") if lse else None
    L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], q, out, scale=scale,
                     window=window, sinks=sinks, lse=ls, workspace=workspace)
    sc = q.shape[2] ** -0.5 if scale is None else scale
    o, rl, amp, big = attention(m["cache"], m["table"], m["qstart"], m["seq"], q, sc, window,
                                sinks)
    compare(out, o, amp, big)
    if lse:
        none = torch.isinf(rl)
        assert torch.equal(torch.isneginf(ls), none)
        d = (ls.double() - rl).abs()[~none]
        assert bool((d <= lse_tolerance(rl, big)[~none]).all()), float(d.max())
    return out


def compare(out, o, amp, big):
    fin = torch.isfinite(o)
    assert torch.equal(torch.isfinite(out), fin), "not finite where it should be, or the reverse"
    assert torch.equal(torch.isnan(out), torch.isnan(o))
    d = (out.double() - o).abs()
    over = (d > tolerance(o, amp, big, out.dtype)) & fin
    assert not bool(over.any()), (
        f"{int(over.sum())} of {over.numel()} off; worst {float(d[fin].max())} at "
        f"{over.nonzero()[0].tolist()}")
