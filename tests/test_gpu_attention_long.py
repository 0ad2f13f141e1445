"""pagedAttention over long contexts of values of one sign, where a bias of the sums would show:
sums that were cut off instead of rounded would all come out low."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
import attention_refs as R  # noqa: E402


def positive(keys, new, requests, x, cache, dim, heads=1):
    """Requests that share one table of `keys` keys, values close to 1, flat weights.  One key
    head: with more requests than CTAs, an item's keys are added up by one or two of them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(keys + dim)
    ps = 64
    pages = -(-keys // ps)
    shape = (pages, ps, 1, dim)
    if cache == "int8":
        k = torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        v = torch.randint(90, 128, shape, generator=g, device="cuda", dtype=torch.int8)
        ks = torch.full(shape[:3], 0.01, device="cuda")
        vs = 0.009 + 0.001 * torch.rand(shape[:3], generator=g, device="cuda")
        c = L.KVCache(k, v, ks, vs)
    else:
        k, v = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
        c = L.KVCache(k.to(R.DT[cache]), (1 + 0.1 * v).to(R.DT[cache]))
    i32 = dict(dtype=torch.int32, device="cuda")
    q = 0.05 * torch.randn(requests * new, heads, dim, generator=g, device="cuda")
    return dict(cache=c, table=torch.arange(pages, **i32)[None].repeat(requests, 1),
                qstart=torch.arange(requests + 1, **i32) * new,
                seq=torch.full((requests,), keys, **i32), q=q.to(R.DT[x]))


def run(m, look, scale=None, window=0):
    """Every request, held to 64 bits in the first `look`: (relative errors, s)."""
    out = torch.full_like(m["q"], math.nan)
    L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out, window=window)
    rows = int(m["qstart"][look])
    o, _, amp, big = R.attention(m["cache"], m["table"][:look], m["qstart"][:look + 1],
                                 m["seq"][:look], m["q"][:rows], m["q"].shape[2] ** -0.5, window)
    assert bool(torch.isfinite(out).all())
    return out[:rows], o, amp, big


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("cache", ["fp16", "bf16", "int8"])
def test_fp32_sums_of_single_tokens_are_rounded(cache, dim):
    """A warp adds up at most n = keys / 64 steps in fp32 (fewer where a step has 32 keys), each
    sum rounded once: errors of at most 2^-24 of the sum, independent of one another, so 5
    sqrt(n) 2^-24 in the numerator and as much in the denominator (5 standard deviations of
    errors that were all at their limit).  Within a step at most 6 products are cut off, each
    by less than 2^-23 of the step's sum, which is all that may show in the mean."""
    keys = 131000
    out, o, amp, big = run(positive(keys, 1, 400, "fp32", cache, dim), 48)
    e = (out.double() - o) / o
    sums = 2 * 5 * math.sqrt(keys / 64) * 2.0 ** -24
    assert bool((e.abs() <= 2.0 ** -19 * (big[..., None] + 1) + sums).all()), float(e.abs().max())
    assert abs(float(e.mean())) <= 2.0 ** -20, float(e.mean())


@pytest.mark.parametrize("x,cache,heads,kv", [("bf16", "bf16", 4, 4), ("fp16", "fp16", 6, 2),
                                              ("bf16", "int8", 2, 2)])
def test_infinities_of_long_items_before_many_short_ones(x, cache, heads, kv):
    """A prompt that fills both row tiles, with infinities that only later rows see, before
    dozens of short requests (one row tile each) with infinities of their own: every row gets
    those that it sees and no others, whichever half of the kernel is ahead."""
    lens = ([(100, 768 * kv // heads)] + [(37 * i % 90, 26 + i % 9) for i in range(39)]) * 12
    m = R.make(40, lens, heads, kv, 64, 16, x, cache)
    c, tab = m["cache"], m["table"]
    clean = L.KVCache(c.k, c.v.clone(), c.kScales,
                      None if c.vScales is None else c.vScales.clone())
    seen = []  # per request: the keys that hold an infinity
    for b, (ctx, new) in enumerate(lens):
        at = [ctx + new - 1, ctx + new // 2, ctx + new // 3] if new > 100 else [ctx + new - 2]
        seen.append(at)
        for j in at:
            where = (int(tab[b, j // 16]), j % 16)
            if cache == "int8":
                c.v[where] = 1
                c.vScales[where] = math.inf
            else:
                c.v[where][:, ::3] = math.inf
                clean.v[where][:, ::3] = 0
            if cache == "int8":
                clean.v[where] = 1
    for _ in range(3):
        out = torch.full_like(m["q"], math.nan)
        L.pagedAttention(c, tab, m["qstart"], m["seq"], m["q"], out)
        if _ == 0:
            first = out
        assert torch.equal(first.isinf(), out.isinf())
        assert torch.equal(torch.where(first.isinf(), 0, first), torch.where(out.isinf(), 0, out))
    hot = torch.zeros(out.shape[0], dtype=torch.bool, device="cuda")
    for b, (ctx, new) in enumerate(lens):
        t0 = int(m["qstart"][b])
        hot[t0 + min(seen[b]) - ctx:t0 + new] = True
    inf = torch.zeros_like(out, dtype=torch.bool)
    inf[hot] = True
    if cache != "int8":
        inf[:, :, [d for d in range(64) if d % 3]] = False
    assert torch.equal(torch.isposinf(out), inf)
    o, _, amp, big = R.attention(clean, tab, m["qstart"], m["seq"], m["q"], 64 ** -0.5)
    ok = ~inf
    d = (out.double() - o).abs()
    assert bool((d <= R.tolerance(o, amp, big, out.dtype))[ok].all())


@pytest.mark.parametrize("x,cache", [("fp16", "fp16"), ("bf16", "fp16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_sums_over_hundreds_of_thousands_of_keys(x, cache, dim):
    """16-bit results take one rounding of the output and one of each weight; what the tensor
    cores' sums are cut off by has to stay well below that: 1024 products of 16 keys, each cut
    by less than 2^-23 of a sum that is half the whole on average."""
    out, o, amp, big = run(positive(300000, 128, 160, x, cache, dim, heads=2), 4)
    tol = R.tolerance(o, amp, big, out.dtype) + 1024 * 2.0 ** -24 * amp
    d = (out.double() - o).abs()
    assert bool((d <= tol).all()), float((d / o).max())


@pytest.mark.parametrize("x,cache,keys,dims", [("fp16", "fp16", 40000, (64, 96, 128)),
                                               ("bf16", "bf16", 280000, (64, 128)),
                                               ("bf16", "int8", 150000, (64,))])
@pytest.mark.parametrize("requests", [1, 42])
def test_long_chunks_whose_maxima_grow(x, cache, keys, dims, requests):
    """Sums that leave tensor memory in parts: keys that grow along the context, so that the
    running maximum moves after each part, items in one CTA and cut between CTAs."""
    for dim in dims:
        m = positive(keys, 100, requests, x, cache, dim, heads=4)
        c = m["cache"]
        g = torch.Generator(device="cuda")
        g.manual_seed(dim)
        sign = torch.randint(0, 2, c.v.shape[:2], generator=g, device="cuda")[..., None, None] * 2 - 1
        c.v.mul_(sign.to(c.v.dtype))
        ramp = torch.linspace(0.2, 3.0, keys // 64 + 1, device="cuda")[:c.pages, None, None]
        if cache == "int8":
            c.kScales.mul_(ramp)
        else:
            c.k.mul_(ramp[..., None].to(c.k.dtype))
        m["q"].mul_(30)
        for window in (0, keys - 3000):
            out, o, amp, big = run(m, min(requests, 2), window=window)
            tol = R.tolerance(o, amp, big, out.dtype) + 2.0 ** -13 * amp
            assert bool(((out.double() - o).abs() <= tol).all())


@pytest.mark.parametrize("x,cache", [("fp16", "fp16"), ("bf16", "fp16"), ("bf16", "bf16"),
                                     ("bf16", "int8")])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_short_requests_in_tables_with_room_for_long_ones(x, cache, dim):
    """The table's width may choose the kernel; the results do not show it."""
    m = R.make(41, [(0, 70), (5, 33), (130, 129), (300, 1), (511, 250)], 4, 2, dim, 16, x, cache,
               tail=math.nan)
    narrow = R.check(m, window=200, sinks=3)
    wide = torch.full((5, 10000), -1, dtype=torch.int32, device="cuda")
    wide[:, :m["table"].shape[1]] = m["table"]
    m["table"] = wide[:, :9000]
    assert torch.equal(R.check(m, window=200, sinks=3), narrow)


@pytest.mark.parametrize("x,cache,dim", [("bf16", "bf16", 128), ("fp32", "fp16", 64),
                                         ("fp32", "int8", 64)])
def test_infinities_everywhere_in_long_contexts_with_holes(x, cache, dim):
    """Every tile is seen in part and holds infinities, in all items at once: what that costs
    stays far from the time after which the kernel's roles give up waiting for one another."""
    keys, requests, new = 600000, 148, 128
    pages = 64
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros(pages, 16, 1, dim, device="cuda", dtype=R.DT[cache])
    v = torch.ones_like(k)
    col = torch.arange(dim, device="cuda") % 4
    if cache == "int8":
        v[..., col == 1] = -1
        v[..., col == 3] = 0
        s = torch.full((pages, 16, 1), math.inf, device="cuda")
        c = L.KVCache(k, v, torch.ones_like(s), s)
        want = torch.tensor([math.inf, -math.inf, math.inf, math.nan], device="cuda")
    else:
        v[..., col == 0] = math.inf
        v[..., col == 1] = -math.inf
        v[:, ::2, :, col == 2] = math.inf
        v[:, 1::2, :, col == 2] = -math.inf
        c = L.KVCache(k, v)
        want = torch.tensor([math.inf, -math.inf, math.nan, 1.0], device="cuda")
    table = torch.randint(0, pages, (requests, keys // 16), **i32)
    table[:, ::3] = -1
    q = torch.zeros(requests * new, 1, dim, device="cuda", dtype=R.DT[x])
    out = torch.full_like(q, 7.0)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    L.pagedAttention(c, table, torch.arange(requests + 1, **i32) * new,
                     torch.full((requests,), keys, **i32), q, out)
    end.record()
    end.synchronize()
    assert L._native.device_error() == 0
    assert torch.allclose(out.float(), want[col].expand_as(out), rtol=2.0 ** -18, atol=0,
                          equal_nan=True)
    assert start.elapsed_time(end) < 1000.0
