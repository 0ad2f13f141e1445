"""assignPages, storeKV and loadKV: exact against plain forms."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
import attention_refs as R  # noqa: E402


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run_assign(ctx, new, ps, free, head, table, tokens, positions=True, stride=0):
    n = len(ctx)
    full = torch.full((n, table.shape[1] + stride), -5, dtype=torch.int32, device="cuda")
    tab = full[:, :table.shape[1]]
    tab.copy_(torch.from_numpy(table))
    qs, seq = i32([-9] * (n + 1)), i32([-9] * n)
    slots = torch.full((tokens,), -9, dtype=torch.int64, device="cuda")
    pos = i32([-9] * tokens) if positions else None
    out = i32([-9])
    L.assignPages(i32(ctx), i32(new), ps, i32(free), i32([head]), tab, qs, seq, slots, pos, out)
    assert bool((full[:, table.shape[1]:] == -5).all())
    return dict(table=tab, qstart=qs, seq=seq, slots=slots, pos=pos, head=out)


def check_assign(ctx, new, ps, spare=4, head=1, tokens=None, width=None, seed=0, **kw):
    rng = np.random.default_rng(seed)
    used = [-(-max(c, 0) // ps) for c in ctx]
    last = [-(-(max(c, 0) + max(n, 0)) // ps) for c, n in zip(ctx, new)]
    width = max(last + [1]) + 2 if width is None else width
    pages = rng.permutation(sum(used) + sum(last) + 50).astype(np.int32)
    table = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for b, u in enumerate(used):
        u = min(u, width)
        table[b, :u] = pages[at:at + u]
        at += u
    free = pages[at:at + max(0, sum(last) - sum(used) + spare + head)].tolist()
    tokens = sum(max(n, 0) for n in new) + 3 if tokens is None else tokens
    got = run_assign(ctx, new, ps, free, head, table, tokens, **kw)
    want = R.assign_pages(ctx, new, ps, free, head, table.copy(), tokens)
    for name, w in want.items():
        if got[name] is not None:
            g = got[name].cpu().numpy().reshape(-1)
            assert np.array_equal(g, np.asarray(w).reshape(-1)), name
    return want


@pytest.mark.parametrize("ps", [1, 7, 16, 128])
@pytest.mark.parametrize("b", [1, 2, 31, 600, 1300])
def test_assign_pages(b, ps):
    rng = np.random.default_rng(b * 1000 + ps)
    ctx = rng.integers(0, 300, b).tolist()
    check_assign(ctx, [1] * b, ps)
    check_assign(ctx, rng.integers(0, 90, b).tolist(), ps, stride=3)


def test_assign_edges():
    check_assign([], [], 16)
    check_assign([0], [0], 16)
    check_assign([0, 16, 15, 17], [16, 0, 1, 31], 16)
    check_assign([0] * 5, [0] * 5, 16)
    check_assign([5, 9], [100000, 1], 16, positions=False)
    check_assign([-3, 4], [2, -8], 16)
    # fewer and more entries in the slot map than tokens
    check_assign([3, 4, 5], [10, 10, 10], 4, tokens=17)
    check_assign([3, 4, 5], [10, 10, 10], 4, tokens=0)
    check_assign([3, 4, 5], [10, 10, 10], 4, tokens=3000)


def test_assign_runs_out_of_pages_and_of_table():
    w = check_assign([30, 3, 40], [40, 40, 40], 8, spare=-7)
    assert -1 in w["slots"][:120]
    w = check_assign([30, 3, 40], [40, 40, 40], 8, width=6)
    assert -1 in w["slots"][:120]
    check_assign([30, 3], [40, 40], 8, spare=-100, head=0)


def test_assign_feeds_itself():
    """Steps in a row: the free head alternates between two tensors."""
    ps, b, width = 4, 3, 30
    free = torch.randperm(90, device="cuda").to(torch.int32)
    heads = [i32([0]), i32([0])]
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    ctx, seen = i32([0, 0, 0]), set()
    for step, new in enumerate([[5, 1, 0], [1, 1, 9], [0, 7, 1], [1, 1, 1]]):
        t = sum(new)
        seq, qs, slots = i32([0] * b), i32([0] * (b + 1)), torch.empty(
            t, dtype=torch.int64, device="cuda")
        L.assignPages(ctx, i32(new), ps, free, heads[step % 2], table, qs, seq, slots, None,
                      heads[1 - step % 2])
        s = slots.tolist()
        assert min(s) >= 0 and not seen & set(s) and len(set(s)) == t
        seen |= set(s)
        ctx = seq
    assert ctx.tolist() == [7, 10, 11]
    assert heads[0].tolist() == [2 + 3 + 3]


ROWS = ["fp32", "fp16", "bf16"]


def expected(x, cache):
    x = x.float().cpu()
    if cache == "int8":
        q, s = R.quantize_rows(x.numpy())
        return torch.from_numpy(q), torch.from_numpy(s)
    return x.to(R.DT[cache]), None


def new_cache(pages, ps, hkv, dim, cache, heads_first=False):
    shape = (pages, hkv, ps, dim) if heads_first else (pages, ps, hkv, dim)
    ts = [torch.zeros(shape, dtype=R.DT[cache], device="cuda") for _ in range(2)]
    if heads_first:
        ts = [t.transpose(1, 2) for t in ts]
    ss = [torch.zeros(pages, ps, hkv, device="cuda") for _ in range(2)] if cache == "int8" else []
    return L.KVCache(*ts, *ss)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.cpu().float(), nan=123.0),
                       torch.nan_to_num(b.cpu().float(), nan=123.0))


@pytest.mark.parametrize("dim", [16, 64, 96, 128, 144, 256])
@pytest.mark.parametrize("cache", ["fp16", "bf16", "int8"])
@pytest.mark.parametrize("x", ROWS)
def test_store_and_load(x, cache, dim):
    for t, hkv, ps, first in ((1, 1, 1, False), (37, 3, 5, False), (300, 2, 16, True)):
        torch.manual_seed(dim + t)
        pages = -(-t // ps) + 2
        c = new_cache(pages, ps, hkv, dim, cache, first)
        k, v = (torch.randn(t, hkv, dim, device="cuda") *
                torch.exp2(torch.randint(-20, 10, (t, hkv, 1), device="cuda").float())
                for _ in range(2))
        k[0, 0] = 0.0
        k, v = k.to(R.DT[x]), v.to(R.DT[x])
        slots = torch.randperm(pages * ps, device="cuda")[:t]
        L.storeKV(c, k, v, slots)
        for rows, pool, sc in ((k, c.k, c.kScales), (v, c.v, c.vScales)):
            want, s = expected(rows, cache)
            assert torch.equal(pool[slots // ps, slots % ps].cpu(), want)
            if s is not None:
                assert torch.equal(sc[slots // ps, slots % ps].cpu(), s)
            # and nothing else was touched
            rest = torch.ones(pages, ps, dtype=torch.bool, device="cuda")
            rest[slots // ps, slots % ps] = False
            assert not pool[rest].any()
        for y in ROWS:
            gk, gv = (torch.full((t, hkv, dim), math.nan, dtype=R.DT[y], device="cuda")
                      for _ in range(2))
            L.loadKV(c, slots, gk, gv)
            for got, rows in ((gk, k), (gv, v)):
                want, s = expected(rows, cache)
                want = want.float() if s is None else want.float() * s[..., None]
                assert same(got, want.to(R.DT[y]))


@pytest.mark.parametrize("cache", ["fp16", "int8"])
def test_slots_outside_the_cache(cache):
    c = new_cache(3, 4, 2, 64, cache)
    k, v = (torch.randn(6, 2, 64, device="cuda") for _ in range(2))
    slots = torch.tensor([-1, 3, 12, 2 ** 40, -2 ** 40, 11], device="cuda")
    L.storeKV(c, k, v, slots)
    want, _ = expected(k, cache)
    assert torch.equal(c.k[0, 3].cpu(), want[1]) and torch.equal(c.k[2, 3].cpu(), want[5])
    assert int((c.k != 0).any(-1).any(-1).sum()) == 2
    gk, gv = (torch.full_like(k, 7.0) for _ in range(2))
    L.loadKV(c, slots, gk, gv)
    assert not gk[[0, 2, 3, 4]].any() and bool(gk[[1, 5]].any())


@pytest.mark.parametrize("cache", ["fp16", "bf16", "int8"])
def test_strided_and_unaligned_rows(cache):
    """Keys and values as slices of packed projections at odd offsets."""
    t, hkv, dim = 21, 2, 96
    for x in ROWS:
        packed = torch.randn(t * 700 + 1, device="cuda").to(R.DT[x])[1:].view(t, 700)
        k = packed[:, 3:3 + hkv * dim].view(t, hkv, dim)
        v = packed[:, 301:301 + hkv * dim].view(t, hkv, dim)
        c = new_cache(4, 8, hkv, dim, cache)
        slots = torch.randperm(32, device="cuda")[:t]
        L.storeKV(c, k, v, slots)
        for rows, pool in ((k, c.k), (v, c.v)):
            assert torch.equal(pool[slots // 8, slots % 8].cpu(), expected(rows, cache)[0])
        before = packed.clone()
        gk, gv = k, v
        L.loadKV(c, slots, gk, gv)
        want, s = expected(before[:, 3:3 + hkv * dim].view(t, hkv, dim), cache)
        want = want.float() if s is None else want.float() * s[..., None]
        assert same(gk, want.to(R.DT[x]))
        before[:, 3:3 + hkv * dim] = packed[:, 3:3 + hkv * dim]
        before[:, 301:301 + hkv * dim] = packed[:, 301:301 + hkv * dim]
        assert torch.equal(packed, before), "wrote outside of the rows"


def test_int8_bytes_are_those_of_calibrate_and_quantize():
    for dim in (64, 96, 128):
        x = torch.randn(50, 2, dim, device="cuda") * 3
        x[3, 1, 5] = math.inf
        x[4, 0, 7] = math.nan
        x[5, 0] = 1e-42
        c = new_cache(4, 16, 2, dim, "int8")
        slots = torch.arange(50, device="cuda")
        L.storeKV(c, x, x, slots)
        s = torch.empty(100, device="cuda")
        q = torch.empty(100 * dim, dtype=torch.int8, device="cuda")
        L.calibrateSymmetric(x.view(-1), dim, 127.0, s)
        L.quantizeBatch(x.view(-1), s, dim, q)
        assert torch.equal(c.k.view(-1, 2, dim)[:50].reshape(-1), q)
        assert torch.equal(c.vScales.view(-1, 2)[:50].reshape(-1), s)


def test_rows_past_2_to_31_elements():
    ps, hkv, d = 16, 8, 128
    pages = 2 ** 31 // (ps * hkv * d) + 5
    pool = torch.zeros(pages, ps, hkv, d, dtype=torch.int8, device="cuda")
    sc = torch.zeros(pages, ps, hkv, device="cuda")
    c = L.KVCache(pool, torch.zeros_like(pool), sc, torch.zeros_like(sc))
    x = torch.randn(3, hkv, d, device="cuda")
    slots = torch.tensor([0, pages * ps - 1, 2 ** 31 // (hkv * d) + 1], device="cuda")
    L.storeKV(c, x, x, slots)
    got = torch.empty_like(x)
    L.loadKV(c, slots, got, torch.empty_like(x))
    want, s = expected(x, "int8")
    assert same(got, want.float() * s[..., None])
    assert int((sc != 0).sum()) == 3 * hkv


def test_empty_calls():
    c = new_cache(2, 4, 1, 64, "fp16")
    e = torch.empty(0, 1, 64, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    L.storeKV(c, e, e, none)
    L.loadKV(c, none, e, e)
    c2 = L.KVCache.allocate(5, 8, 2, 64, torch.int8)
    assert c2.pages == 5 and c2.pageSize == 8 and c2.kvHeads == 2 and c2.headDim == 64
    x = torch.randn(7, 2, 64, device="cuda")
    L.storeKV(c2, x, x, torch.arange(7, device="cuda"))
    got = torch.empty_like(x)
    L.loadKV(c2, torch.arange(7, device="cuda"), got, torch.empty_like(x))
    want, s = expected(x, "int8")
    assert same(got, want.float() * s[..., None])


def test_assign_arrays_side_by_side():
    """Arrays that touch, and one between the rows of the table, are taken; lengths updated in
    place are not."""
    ctx, new, ps, free = [5, 0, 31, 16], [3, 40, 1, 0], 8, list(range(20, 5, -1))
    n, tokens, width = len(ctx), sum(new) + 2, 7
    buf = torch.full((400,), -1, dtype=torch.int32, device="cuda")
    at = [0]

    def take(k, values=()):
        t = buf[at[0]:at[0] + k]
        at[0] += k
        if values:
            t.copy_(i32(list(values)))
        return t
    c, a, f, head = take(n, ctx), take(n, new), take(len(free), free), take(1, [1])
    seq, qs, pos = take(n), take(n + 1), take(tokens)
    take(at[0] % 2)
    slots = take(2 * tokens).view(torch.int64)
    rows = take(n * (width + 3)).view(n, width + 3)
    table, out = rows[:, :width], rows[1, width:width + 1]
    start = np.full((n, width), -1, np.int32)
    for b, x in enumerate(ctx):
        start[b, :-(-x // ps)] = 30 + b
    table.copy_(torch.from_numpy(start))
    want = R.assign_pages(ctx, new, ps, free, 1, start.copy(), tokens)
    L.assignPages(c, a, ps, f, head, table, qs, seq, slots, pos, out)
    for name, got in dict(table=table, qstart=qs, seq=seq, slots=slots, pos=pos, head=out).items():
        assert np.array_equal(got.cpu().numpy().reshape(-1), np.asarray(want[name]).reshape(-1)), name
    assert c.tolist() == ctx and a.tolist() == new and f.tolist() == free and head.tolist() == [1]
    for wrong in (dict(seq=c), dict(seq=a), dict(out=head), dict(qs=buf[n - 1:2 * n])):
        k = {**dict(seq=seq, qs=qs, out=out), **wrong}
        with pytest.raises(L._native.NativeError):
            L.assignPages(c, a, ps, f, head, table, k["qs"], k["seq"], slots, pos, k["out"])


@pytest.mark.parametrize("head", [4, 5, 9])
def test_assign_from_the_end_of_the_free_list(head):
    """A head at or past the end of the list gives no page, and the next one is its end."""
    ctx, new, ps = [3, 8], [9, 1], 4
    table = np.full((2, 6), -1, np.int32)
    table[0, 0], table[1, :2] = 11, (12, 13)
    want = R.assign_pages(ctx, new, ps, [7, 6, 5, 4], head, table.copy(), 12)
    got = run_assign(ctx, new, ps, [7, 6, 5, 4], head, table, 12)
    for name, w in want.items():
        assert np.array_equal(got[name].cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name
