"""pagedAttention against the 64-bit form: types, head layouts, lengths, pages, windows and
sinks, rows that see nothing, and what masked places hold."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
from nim_lowprec_b200 import _native as N  # noqa: E402
import attention_refs as R  # noqa: E402

PAIRS = [("fp32", "fp16"), ("fp32", "bf16"), ("fp32", "int8"), ("fp16", "fp16"),
         ("fp16", "bf16"), ("fp16", "int8"), ("bf16", "fp16"), ("bf16", "bf16"),
         ("bf16", "int8")]
DECODE = [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (31, 1), (200, 1), (777, 1)]
CHUNK = [(0, 1), (0, 70), (5, 33), (130, 129), (300, 1), (511, 250)]


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("x,cache", PAIRS)
def test_decode_types(x, cache, dim):
    R.check(R.make(1, DECODE, 8, 2, dim, 16, x, cache))


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("x,cache", PAIRS)
def test_chunk_types(x, cache, dim):
    R.check(R.make(2, CHUNK, 4, 2, dim, 16, x, cache))


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (6, 2), (7, 1), (8, 1), (9, 1), (16, 1),
                                      (24, 8), (32, 32)])
@pytest.mark.parametrize("lens", [DECODE, CHUNK], ids=["decode", "chunk"])
def test_head_layouts(heads, kv, lens):
    R.check(R.make(3, lens, heads, kv, 64, 16, "fp16", "fp16"))


@pytest.mark.parametrize("ps", [1, 3, 8, 16, 24, 64, 300])
@pytest.mark.parametrize("x,cache", [("fp32", "int8"), ("bf16", "bf16")])
@pytest.mark.parametrize("lens", [DECODE, CHUNK], ids=["decode", "chunk"])
def test_page_sizes(ps, x, cache, lens):
    R.check(R.make(4, lens, 6, 2, 128, ps, x, cache, tail=math.nan))


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (40, 3), (128, 200), (500, 16),
                                          (5000, 4), (33, 1)])
@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("fp32", "int8"), ("bf16", "bf16")])
@pytest.mark.parametrize("lens", [DECODE, CHUNK], ids=["decode", "chunk"])
def test_windows_and_sinks(window, sinks, x, cache, lens):
    R.check(R.make(5, lens, 4, 2, 64, 16, x, cache), window=window, sinks=sinks)


def test_long_window_edges():
    m = R.make(6, [(3000, 600), (2047, 1), (100, 2000)], 4, 2, 128, 32, "bf16", "bf16")
    R.check(m, window=1024, sinks=4)
    R.check(m, window=1000, sinks=130)


@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("fp32", "int8"), ("bf16", "bf16")])
@pytest.mark.parametrize("lens", [[(40000, 1)], [(30001, 40)], [(9000, 1), (3, 1), (70000, 1)]],
                         ids=["one", "chunk", "ragged"])
def test_long_contexts(x, cache, lens):
    R.check(R.make(7, lens, 8, 2, 128, 64, x, cache))


@pytest.mark.parametrize("lens", [[(0, 1)] * 700, [(i % 50, 1 + i % 3) for i in range(600)]],
                         ids=["one token", "short"])
def test_many_requests(lens):
    R.check(R.make(8, lens, 4, 4, 64, 16, "fp32", "fp16"))


def test_long_chunk_in_every_type():
    for x, cache in PAIRS:
        R.check(R.make(9, [(100, 1100)], 8, 2, 128, 16, x, cache))


def test_requests_without_new_tokens():
    R.check(R.make(10, [(5, 0), (20, 1), (0, 0), (0, 3), (400, 0)], 4, 2, 64, 16))
    R.check(R.make(10, [(5, 0), (20, 100), (0, 0), (0, 300), (400, 0)], 4, 2, 64, 16))


@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "int8")])
@pytest.mark.parametrize("n", [3, 90])
def test_rows_that_see_nothing(x, cache, n):
    """Requests shorter than their new tokens (the first tokens lie before position 0), and a
    table without pages."""
    m = R.make(11, [(40, n), (20, n), (50, n)], 4, 2, 64, 16, x, cache)
    m["seq"][0] = n - 2
    m["seq"][1] = 0
    m["table"][2] = -1
    out = R.check(m)
    assert not out[:2].any() and not out[n:].any()


@pytest.mark.parametrize("n", [1, 70])
def test_missing_and_bad_pages_are_not_seen(n):
    """Holes in a table, as a window leaves them, and entries outside the cache."""
    for x, cache in (("fp32", "int8"), ("bf16", "bf16")):
        m = R.make(12, [(200, n), (333, n)], 4, 2, 64, 16, x, cache)
        m["table"][0, 2:5] = -1
        m["table"][1, 0] = m["cache"].pages
        m["table"][1, 3] = -7
        m["table"][1, 7] = 2 ** 31 - 1
        R.check(m)
        R.check(m, window=60, sinks=20)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("fp16", "fp16"), ("bf16", "bf16"),
                                     ("fp32", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("lens,window", [([(37, 1), (5, 1)], 0), ([(37, 60), (5, 90)], 0),
                                         ([(300, 200), (90, 1)], 50)])
def test_masked_places_may_hold_anything(bad, x, cache, lens, window):
    """Page tails, pages of nobody, and keys that only later tokens see or only earlier ones."""
    m = R.make(13, lens, 4, 2, 64, 16, x, cache, tail=bad)
    c, tab = m["cache"], m["table"]
    at = sum(lens[0]) - 1  # request 0's last key: its own row alone sees it
    where = (int(tab[0, at // 16]), at % 16)
    if cache == "int8":
        c.vScales[where] = bad
    else:
        c.v[where] = bad
    out = R.check(m, window=window, sinks=4 if window else 0)
    last = int(m["qstart"][1]) - 1
    assert bool(torch.isfinite(out[:last]).all()) and bool(torch.isfinite(out[last + 1:]).all())
    assert not bool(torch.isfinite(out[last]).all())


@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("bf16", "bf16"), ("fp32", "int8"),
                                     ("bf16", "int8")])
@pytest.mark.parametrize("n", [3, 100])
def test_bad_values_among_many_partly_seen_tiles(x, cache, n):
    """More tiles with holes and bad values than are noted one by one."""
    m = R.make(22, [(9000, n)], 2, 1, 64, 16, x, cache)
    c = m["cache"]
    m["table"][0, 3::8] = -1
    pages = m["table"][0, 1::8].long()
    pages = pages[(pages >= 0)][:-2]
    if cache == "int8":
        c.vScales[pages, 5] = math.inf
    else:
        c.v[pages, 5] = math.inf
    out = torch.empty_like(m["q"])
    L.pagedAttention(c, m["table"], m["qstart"], m["seq"], m["q"], out)
    assert not bool(torch.isfinite(out).any())
    # and one that only the last row sees, far from them
    c.v[:] = 1
    if cache == "int8":
        c.vScales[:] = 1.0
    last = 9000 + n - 1
    at = (int(m["table"][0, last // 16]), last % 16)
    if cache == "int8":
        c.vScales[at] = math.nan
    else:
        c.v[at] = math.nan
    L.pagedAttention(c, m["table"], m["qstart"], m["seq"], m["q"], out)
    assert bool(torch.isfinite(out[:-1]).all()) and not bool(torch.isfinite(out[-1]).any())
    assert bool(((out[:-1].float() - 1).abs() < 0.01).all())


def test_a_cache_full_of_nan_stays_so():
    for x, cache in (("fp32", "fp16"), ("bf16", "bf16")):
        m = R.make(23, [(700, 300), (50, 1)], 4, 2, 128, 16, x, cache)
        m["cache"].v[:] = math.nan
        out = torch.zeros_like(m["q"])
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out, window=200)
        assert bool(torch.isnan(out).all())


def test_seen_nan_key_and_infinite_scores():
    m = R.make(14, [(64, 1), (64, 40)], 2, 2, 64, 16, "fp32", "fp16")
    m["cache"].k[int(m["table"][0, 1]), 3] = math.nan
    m["cache"].k[int(m["table"][1, 4]), 5] = math.nan  # position 69: new token 5 and later
    out = torch.empty_like(m["q"])
    L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out)
    assert bool(torch.isnan(out[0]).all())
    assert bool(torch.isfinite(out[1:6]).all()) and bool(torch.isnan(out[6:]).all())


@pytest.mark.parametrize("x,cache", [("fp32", "fp16"), ("fp32", "int8"), ("bf16", "bf16")])
@pytest.mark.parametrize("n", [1, 80])
def test_large_and_tiny_queries(x, cache, n):
    """Rows of very different size in one tile, sharp and flat softmaxes, a zero row."""
    m = R.make(15, [(500, n), (31, n)], 4, 2, 128, 16, x, cache)
    f = torch.tensor([1e-30, 1e-4, 1.0, 30.0, 0.0, 1e-38], device="cuda")
    i = torch.arange(m["q"].shape[0] * 4, device="cuda") % 6
    m["q"] = (m["q"].float() * f[i].reshape(-1, 4, 1)).to(m["q"].dtype)
    R.check(m)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(scale):
    R.check(R.make(16, [(90, 1), (200, 40)], 4, 2, 64, 16), scale=scale)


@pytest.mark.parametrize("n", [1, 100])
def test_strides_and_alignment(n):
    """Queries as a slice of packed rows at an odd offset, output with heads outside of tokens,
    a cache with heads outside of tokens, a table that is a slice."""
    for x, cache in (("fp32", "fp16"), ("fp16", "int8"), ("bf16", "bf16")):
        m = R.make(17, [(70, n), (20, n)], 4, 2, 64, 16, x, cache, heads_first=True)
        q = m["q"]
        t = q.shape[0]
        packed = torch.randn(t * 4 * 200 + 1, device="cuda").to(q.dtype)
        view = packed[1:].view(t, 4, 200)[:, :, 3:67]
        view.copy_(q)
        m["q"] = view
        wide = torch.full((2, m["table"].shape[1] + 5), 99999, dtype=torch.int32, device="cuda")
        wide[:, 2:-3] = m["table"]
        m["table"] = wide[:, 2:-3]
        hold = torch.full((4, t + 2, 67), 7.0, dtype=q.dtype, device="cuda")
        out = hold[:, 1:-1, 1:65].transpose(0, 1)
        R.check(m, out=out)
        hold[:, 1:-1, 1:65] = 7.0
        assert bool((hold == 7.0).all()), "wrote outside of out"


def test_rows_outside_every_request_are_left_alone():
    m = R.make(18, [(9, 2), (0, 1)], 2, 1, 64, 16)
    for pad in (1, 200):
        q = torch.cat([m["q"], torch.randn(pad, 2, 64, device="cuda")])
        out = torch.full_like(q, 7.0)
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], q, out)
        assert bool((out[3:] == 7.0).all())
        R.compare(out[:3], *(R.attention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"],
                                         64 ** -0.5)[i] for i in (0, 2, 3)))


def test_same_bits_again_and_on_another_stream():
    for lens in ([(5000, 1), (17, 1)], [(700, 500)]):
        m = R.make(19, lens, 8, 2, 128, 16, "bf16", "bf16")
        first = R.check(m)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            outs = [torch.empty_like(first) for _ in range(5)]
            for o in outs:
                L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], o)
        side.synchronize()
        assert all(torch.equal(o, first) for o in outs)


def test_graph_replay_follows_the_lengths():
    """A captured call reads lengths and tables at replay: decode steps of one graph."""
    m = R.make(20, [(900, 1), (33, 1), (64, 1)], 8, 2, 64, 16)
    out, ws = torch.empty_like(m["q"]), L.attentionWorkspace()
    L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out, workspace=ws)
    for lens in ([901, 34, 65], [1, 1, 1], [400, 2, 17]):
        m["seq"].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(math.nan)
        g.replay()
        o, _, amp, big = R.attention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"],
                                     64 ** -0.5)
        R.compare(out, o, amp, big)


def test_cache_past_2_to_31_elements():
    """Rows whose element offset needs more than 32 bits."""
    ps, hkv, d = 16, 8, 128
    pages = 2 ** 31 // (ps * hkv * d) + 40
    k = torch.zeros(pages, ps, hkv, d, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.rand(pages, ps, hkv, device="cuda") + 0.01 for _ in range(2))
    hi = slice(pages - 40, pages)
    for t in (k, v):
        t[hi] = torch.randint(-128, 128, t[hi].shape, device="cuda", dtype=torch.int8)
    cache = L.KVCache(k, v, ks, vs)
    table = torch.arange(pages - 40, pages, device="cuda").to(torch.int32)[None].contiguous()
    low = L.KVCache(k[hi].clone(), v[hi].clone(), ks[hi].clone(), vs[hi].clone())
    for n in (1, 90):
        q = torch.randn(n, 16, d, device="cuda")
        qs, sl = (torch.tensor(z, dtype=torch.int32, device="cuda") for z in ([0, n], [630]))
        outs = [torch.empty_like(q) for _ in range(2)]
        L.pagedAttention(cache, table, qs, sl, q, outs[0])
        L.pagedAttention(low, table - (pages - 40), qs, sl, q, outs[1])
        assert torch.equal(*outs)


def test_queued_gemvs_run_before_the_attention_that_reads_them():
    """Inside a batch the projections are queued; the attention call launches them first."""
    m = R.make(21, [(50, 1)], 2, 1, 64, 16, "fp32", "int8")
    K = 256
    w = torch.randn(128 * K, device="cuda") * 0.05
    s = torch.empty(128 * K // 32, device="cuda")
    L.calibrateSymmetric(w, 32, 7.0, s)
    packed = torch.empty(128 * K // 2, dtype=torch.uint8, device="cuda")
    L.quantizeI4Packed(w, s, 32, packed)
    x = torch.randn(K, device="cuda")
    q = torch.zeros(1, 2, 64, device="cuda")
    out = torch.empty_like(q)
    with L.batch():
        L.quantizeDequantGemvI4Q8(packed, s, 32, x, q.view(-1))
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], q, out)
    m["q"] = q
    R.check(m, out=out.clone())
    assert torch.equal(R.check(m), out)


def test_no_device_error():
    torch.cuda.synchronize()
    assert N.device_error() == 0


def test_python_refusals():
    m = R.make(24, [(9, 2), (0, 1)], 4, 2, 64, 16)
    c, tab, qs, seq, q = m["cache"], m["table"], m["qstart"], m["seq"], m["q"]
    out = torch.empty_like(q)

    def call(cache=c, tab=tab, qs=qs, seq=seq, q=q, out=out, **kw):
        L.pagedAttention(cache, tab, qs, seq, q, out, **kw)
    for kw, error in (
            (dict(q=q.double()), TypeError), (dict(q=q.cpu()), TypeError),
            (dict(out=out.half()), N.NativeError), (dict(seq=seq.long()), TypeError),
            (dict(qs=qs[:-1].clone()), AssertionError), (dict(tab=tab[:1]), AssertionError),
            (dict(tab=tab.long()), TypeError), (dict(tab=tab.t().contiguous().t()), ValueError),
            (dict(q=q[:, :3], out=out[:, :3]), AssertionError), (dict(q=q[0]), AssertionError),
            (dict(q=q[:, :, ::2]), AssertionError), (dict(window=-1), AssertionError),
            (dict(window=1.5), TypeError), (dict(scale="x"), TypeError),
            (dict(scale=math.nan), N.NativeError),
            (dict(lse=torch.empty(3, 4, device="cuda").half()), TypeError),
            (dict(lse=torch.empty(2, 4, device="cuda")), AssertionError),
            (dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")), AssertionError),
            (dict(workspace=torch.zeros(64, device="cuda")), TypeError),
            (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), ValueError)):
        with pytest.raises(error):
            call(**kw)
    k = torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda")
    s = torch.zeros(2, 16, 1, device="cuda")
    for args, error in (((k.float(), k.float()), TypeError), ((k, k.bfloat16()), TypeError),
                        ((k.to(torch.int8),) * 2, TypeError), ((k, k, s, s), TypeError),
                        ((k[0], k[0]), AssertionError), ((k, k[:1]), AssertionError),
                        ((k.to(torch.int8),) * 2 + (s, s[:1]), AssertionError),
                        ((k[..., ::2], k[..., ::2]), ValueError),
                        ((k.to(torch.int8),) * 2 + (s, s.half()), TypeError)):
        with pytest.raises(error):
            L.KVCache(*args)
    odd = torch.zeros(4, 16, 1, 200, dtype=torch.float16, device="cuda")
    with pytest.raises(N.NativeError):  # rows off their 16-byte boundaries
        call(cache=L.KVCache(odd[..., 1:65], odd[..., 1:65]), q=q[:, :1], out=out[:, :1])
    x = torch.zeros(3, 1, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    cc = L.KVCache(k, k.clone())
    for args, error in (((x, x[:2], slots), AssertionError), ((x, x, slots[:2]), AssertionError),
                        ((x, x.half(), slots), N.NativeError), ((x, x, slots.int()), TypeError),
                        ((x[..., :32], x, slots), AssertionError)):
        with pytest.raises(error):
            L.storeKV(cc, *args)


def test_a_capture_without_a_workspace_is_refused():
    m = R.make(25, [(9, 1)], 2, 1, 64, 16)
    out = torch.empty_like(m["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    L.attention._workspaces.pop((0, side.cuda_stream), None)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(g, stream=side):
            out.zero_()
            L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out)
    torch.cuda.synchronize()
    R.check(m)


def test_a_capture_after_calls_on_its_stream_is_refused_without_a_workspace():
    """The workspace that such calls left behind belongs to the stream, not to a graph that may
    be replayed beside it."""
    m = R.make(26, [(300, 1)], 4, 2, 64, 16)
    out = torch.empty_like(m["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(g, stream=side):
            out.zero_()
            L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out)
    torch.cuda.synchronize()
    R.check(m)


def test_graphs_with_workspaces_of_their_own_run_side_by_side():
    m = R.make(27, [(9000, 1), (300, 40), (7000, 1)], 8, 2, 128, 16, "bf16", "bf16")
    first = R.check(m)
    capture, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    outs, spaces, graphs = [], [], []
    for _ in streams:
        outs.append(torch.zeros_like(first))
        spaces.append(L.attentionWorkspace())
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=capture):
            for _ in range(20):
                L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], outs[-1],
                                 workspace=spaces[-1])
    for _ in range(5):
        for s, g, o in zip(streams, graphs, outs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o.fill_(math.nan)
                g.replay()
        eager = torch.empty_like(first)
        L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, first) and all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("x,cache", PAIRS)
def test_infinities_that_every_row_sees(x, cache, dim, n):
    """Values that are not finite in tiles that all rows see whole, at lengths that end with a
    tile: each column has the sum that the definition gives, an infinity or a NaN."""
    m = R.make(28, [(128 - n, n), (320 - n, n), (500, n)], 4, 2, dim, 16, x, cache)
    c = m["cache"]
    if cache == "int8":  # (fp16 results are not to overflow)
        c.vScales.clamp_(max=100.0)
    col = torch.arange(dim, device="cuda") % 8
    for b, (i, j) in enumerate([(5, 21), (0, 17), (7, 37)]):  # keys that are seen by all rows
        first, second = ((int(m["table"][b, k // 16]), k % 16) for k in (i, j))
        if cache == "int8":
            c.vScales[first] = (math.inf, -math.inf, math.nan)[b]
            if b == 1:  # codes of one sign against the other's infinity
                c.vScales[second] = math.inf
            continue
        c.v[first][:, col == 0] = math.inf
        c.v[first][:, col == 1] = -math.inf
        c.v[first][:, col == 2] = math.inf
        c.v[second][:, col == 2] = -math.inf
        c.v[second][:, col == 3] = math.nan
        c.v[second][:, col == 4] = math.inf
    R.check(m)


def test_rows_of_nan_beside_infinities():
    """A NaN in a query makes its row NaN and leaves the others what they are."""
    for n in (1, 90):
        for x, cache in (("fp32", "fp16"), ("fp32", "int8"), ("bf16", "bf16")):
            m = R.make(29, [(128 - n, n), (320 - n, n)], 4, 2, 64, 16, x, cache)
            if cache == "int8":
                m["cache"].vScales[int(m["table"][1, 0]), 3] = math.inf
            else:
                m["cache"].v[int(m["table"][1, 0]), 3] = math.inf
            out = torch.empty_like(m["q"])
            L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], out)
            m["q"][n, 1, 7] = math.nan
            got = R.torch.empty_like(out)
            L.pagedAttention(m["cache"], m["table"], m["qstart"], m["seq"], m["q"], got)
            assert bool(torch.isnan(got[n, 1]).all())
            got[n, 1] = out[n, 1]
            assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(out, nan=7.0))
