"""The cases in which the operators of a sparse feed-forward layer over 8-bit rows are measured: the
norm that makes the rows (addRmsNorm), the router (routeExperts), the experts' products over MXFP4
or MXFP8 weights (expertGemmGated, expertGemm), the sum of a token's experts (combineExperts), and
the rows' own codec (quantizeRows, dequantizeRows).

`run` computes each one in a plain form, with elementary torch operations in fp32; with `own` set,
through the calls that a user makes of nim_lowprec_b200.  8-bit rows are returned as the values that
they stand for, in bf16, which holds every value of an MXFP8 row.
"""
import math
import random

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ cases

def listed():
    return [
        # before the int8 products of a decode step: a handful of tokens (latency)
        dict(name="norm int8 5", op="norm", tokens=5, dim=4096, x="fp32", rows="int8", group=32),
        # before the experts of a prompt: residual stream, 8-bit rows, and rows for the router
        dict(name="norm mx8 8192", op="norm", tokens=8192, dim=4096, x="bf16", rows="mx8", group=32),
        # a decode step's choices
        dict(name="route 13", op="route", tokens=13, experts=64, k=6, pads=0, renorm=True),
        # a padded batch of prompts over many experts
        dict(name="route 8192", op="route", tokens=8192, experts=128, k=8, pads=411, renorm=True),
        # one token: the chosen experts' gate and up matrices are read once
        dict(name="gated 1", op="gated", tokens=1, experts=64, k=8, dim=2048, inner=1408, w="mx4"),
        # a served batch over few large experts: every expert's weights are read
        dict(name="gated 57", op="gated", tokens=57, experts=8, k=2, dim=4096, inner=14336, w="mx4"),
        # a prompt over many small experts
        dict(name="gated 8192", op="gated", tokens=8192, experts=64, k=8, dim=2048, inner=1408,
             w="mx4"),
        # ragged rows of a middle-sized batch, an inner dimension that ends inside a tile
        dict(name="down 300", op="down", tokens=300, experts=128, k=8, dim=2880, inner=736, w="mx4",
             y="bf16"),
        # a prompt's way back to the hidden dimension over 8-bit weights
        dict(name="down 4096", op="down", tokens=4096, experts=8, k=2, dim=4096, inner=14336,
             w="mx8", y="bf16"),
        # one projection of one token, fp32 in and out
        dict(name="linear 1", op="linear", tokens=1, dim=4096, inner=11008, w="mx4", x="fp32",
             y="fp32"),
        # the same kind of projection for a prompt
        dict(name="linear 1000", op="linear", tokens=1000, dim=4096, inner=14336, w="mx8", x="bf16",
             y="fp16"),
        # the layer as a whole, for a step that mixes prompts and single tokens
        dict(name="layer 700", op="layer", tokens=700, experts=32, k=4, dim=2880, inner=1440,
             w="mx4"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "gated", "gated", "down", "down", "linear", "linear", "layer"])
    if op == "norm":
        dim = 32 * _log(rng, 16, 256)
        rows = rng.choice(["mx8", "mx8", "int8"])
        group = rng.choice([32, 64, 128]) if rows == "int8" else 32
        dim = max(group, dim // group * group)
        return dict(op=op, tokens=_log(rng, 1, min(8192, 8192 * 4096 // dim)), dim=dim,
                    x=rng.choice(["fp32", "fp16", "bf16", "bf16"]), rows=rows, group=group)
    if op == "route":
        tokens, experts = _log(rng, 1, 8192), rng.choice([8, 16, 60, 64, 100, 128])
        return dict(op=op, tokens=tokens, experts=experts, k=rng.choice([1, 2, 4, 6, 8]),
                    pads=rng.choice([0, 0, tokens // 7]), renorm=rng.choice([True, True, False]))
    if op == "linear":
        dim, inner = 32 * _log(rng, 16, 350), _log(rng, 500, 14336)
        return dict(op=op, tokens=_log(rng, 1, 2000), dim=dim, inner=inner,
                    w=rng.choice(["mx4", "mx4", "mx8"]), x=rng.choice(["fp32", "fp16", "bf16"]),
                    y=rng.choice(["fp32", "fp16", "bf16"]))
    experts, dim, inner = rng.choice([4, 8, 20, 32, 64, 128]), 32 * _log(rng, 24, 128), \
        32 * _log(rng, 16, 448)
    inner = max(256, min(inner, (8 * 4096 * 14336 // (experts * dim)) // 32 * 32))
    k = rng.choice([1, 2, 4, 6, 8])
    k = min(k, experts)
    most = min(8192, int(3.7e11 / (4 * k * dim * inner)))
    case = dict(op=op, tokens=_log(rng, 1, most), experts=experts, k=k, dim=dim, inner=inner,
                w=rng.choice(["mx4", "mx4", "mx8"]))
    if op == "down":
        case["y"] = rng.choice(["bf16", "bf16", "fp16"])
    return case


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _weights(g, experts, m, k, kind):
    """Normal weights, encoded: MXFP4 as packed codes and fp32 scales (the low nibble is the even
    column), MXFP8 as e4m3 codes and the scales' exponents in a byte."""
    emax = 2 if kind == "mx4" else 8
    scales = torch.empty(experts, m, k // 32, device="cuda")
    if kind == "mx4":
        codes = torch.empty(experts, m, k // 2, dtype=torch.uint8, device="cuda")
        edges = torch.tensor([(a + b) / 2 for a, b in zip(_E2M1, _E2M1[1:])], device="cuda")
    else:
        codes = torch.empty(experts, m, k, dtype=torch.float8_e4m3fn, device="cuda")
    for e in range(experts):
        w = (_randn(g, m, k) * 0.02).reshape(m, k // 32, 32)
        exp = torch.frexp(w.abs().amax(-1)).exponent - 1 - emax
        s = torch.ldexp(torch.ones_like(w[..., 0]), exp)
        scales[e] = s
        w = w / s[..., None]
        if kind == "mx4":
            n = torch.bucketize(w.abs().clamp(max=6.0), edges).to(torch.uint8)
            n = (n + 8 * (w < 0).to(torch.uint8)).reshape(m, k)
            codes[e] = n[:, 0::2] + 16 * n[:, 1::2]
        else:
            codes[e] = w.clamp(-448.0, 448.0).reshape(m, k).to(torch.float8_e4m3fn)
    if kind == "mx8":
        scales = (torch.frexp(scales).exponent + 126).to(torch.uint8)
    return codes, scales


def _logits(g, tokens, experts, pads):
    # some experts are wanted more often than others
    l = 1.5 * _randn(g, tokens, experts) + 0.5 * _randn(g, experts)
    if pads:  # rows that pad the batch see no expert
        l[torch.randperm(tokens, generator=g, device="cuda")[:pads]] = -math.inf
    return l


def _mx8_rows(x):
    """8-bit rows as a program holds them: e4m3 codes, and exponents + 127 in a byte."""
    t, k = x.shape
    b = x.reshape(t, k // 32, 32)
    exp = (torch.frexp(b.abs().amax(-1)).exponent - 9).clamp(-127, 127)
    codes = (b / torch.ldexp(torch.ones_like(b[..., 0]), exp)[..., None]).clamp(-448.0, 448.0)
    return codes.reshape(t, k).to(torch.float8_e4m3fn), (exp + 127).to(torch.uint8)


def _empty_rows(t, k, kind="mx8", group=32):
    if kind == "int8":
        return (torch.zeros(t, k, dtype=torch.int8, device="cuda"),
                torch.zeros(t, k // group, device="cuda"))
    return (torch.zeros(t, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            torch.zeros(t, k // 32, dtype=torch.uint8, device="cuda"))


def _empty_routing(tokens, k, experts):
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(weights=torch.zeros(tokens, k, device="cuda"),
                experts=torch.zeros(tokens, k, **i32), offsets=torch.zeros(experts + 1, **i32),
                row_token=torch.full((tokens * k,), -1, **i32),
                places=torch.zeros(tokens, k, **i32))


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    op, t = case["op"], case["tokens"]
    if op in ("norm", "layer"):
        # the residual stream, where a few channels are large, and what a layer adds to it
        n, xdt = case["dim"], _DT[case.get("x", "bf16")]
        ch = 1.0 + 9.0 * (torch.rand(n, generator=g, device="cuda") > 0.98)
        st.update(x=_randn(g, t, n).to(xdt), res=(2.0 * ch * _randn(g, t, n)).to(xdt),
                  norm=(1.0 + 0.1 * _randn(g, n)).to(xdt), eps=1e-5)
        st["total"] = torch.empty_like(st["x"])
    if op in ("route", "layer", "gated", "down"):
        st["logits"] = _logits(g, t, case["experts"], case.get("pads", 0))
        st["r"] = _empty_routing(t, case["k"], case["experts"])
        st["renorm"] = case.get("renorm", True)
    if op in ("layer", "gated", "down"):
        r = _route_plain(st)
        st["most"] = int((r["offsets"][1:] - r["offsets"][:-1]).max())  # for the plain form's padding
        if op != "layer":
            st["r"] = r
    if op == "norm":
        st["y"] = torch.empty_like(st["x"])
        st["rows"] = _empty_rows(t, case["dim"], case["rows"], case["group"])
        st["vals"] = torch.empty(t, case["dim"], dtype=torch.bfloat16, device="cuda")
        return st
    if op == "route":
        return st
    dim, inner = case["dim"], case["inner"]
    if op in ("gated", "layer"):
        st["up"] = _weights(g, case["experts"], 2 * inner, dim, case["w"])
    if op in ("down", "layer"):
        st["down"] = _weights(g, case["experts"], dim, inner, case["w"])
    if op == "gated":
        st["codes"], st["scales"] = _mx8_rows(_randn(g, t, dim))
        st["vals"] = torch.empty(t * case["k"], inner, dtype=torch.bfloat16, device="cuda")
        st["rows"] = _empty_rows(t * case["k"], inner)
    elif op == "down":
        # a gated hidden layer's values: products of two
        st["codes"], st["scales"] = _mx8_rows(_randn(g, t * case["k"], inner)
                                              * _randn(g, t * case["k"], inner))
        ydt = _DT[case["y"]]
        st["out_rows"] = torch.empty(t * case["k"], dim, dtype=ydt, device="cuda")
        st["out"] = torch.empty(t, dim, dtype=ydt, device="cuda")
    elif op == "linear":
        st["x"] = _randn(g, t, dim).to(_DT[case["x"]])
        st["w"] = _weights(g, 1, inner, dim, case["w"])
        st["rows"] = _empty_rows(t, dim)
        st["offsets"] = torch.tensor([0, t], dtype=torch.int32, device="cuda")
        st["out"] = torch.empty(t, inner, dtype=_DT[case["y"]], device="cuda")
    else:
        st["rows"] = _empty_rows(t, dim)
        st["hidden"] = _empty_rows(t * case["k"], inner)
        st["out_rows"] = torch.empty(t * case["k"], dim, dtype=torch.bfloat16, device="cuda")
        st["out"] = torch.empty(t, dim, dtype=torch.bfloat16, device="cuda")
    if own:
        import nim_lowprec_b200 as L
        for name in ("up", "down", "w"):
            if name in st:
                st[name] = L.ExpertWeights(*st[name], gated=name == "up")
    return st


# ------------------------------------------------------------------ one pass

def run(state):
    return _OPS[state["case"]["op"]][bool(own)](state)


def _norm_own(s):
    import nim_lowprec_b200 as L
    L.addRmsNorm(s["x"], s["res"], s["norm"], s["eps"], total=s["total"], y=s["y"],
                 codes=s["rows"][0], scales=s["rows"][1])
    L.dequantizeRows(*s["rows"], s["vals"])
    return dict(total=s["total"], y=s["y"], vals=s["vals"])


def _norm_values(s):
    """The residual stream after the addition, in its type, and its normed rows in fp32."""
    total = (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    r = total.float()
    mean = r.double().square().mean(-1, keepdim=True)  # a long sum
    return total, r * torch.rsqrt(mean + s["eps"]).float() * s["norm"].float()


def _norm_plain(s):
    c = s["case"]
    total, n = _norm_values(s)
    return dict(total=total, y=n.to(s["x"].dtype), vals=_quantized(n, c["rows"], c["group"]).bfloat16())


def _quantized(x, kind, group=32):
    """The values that 8-bit rows of x stand for."""
    b = x.reshape(x.shape[0], -1, group)
    amax = b.abs().amax(-1, keepdim=True)
    if kind == "int8":
        scale = torch.where(amax == 0, torch.ones_like(amax), amax / torch.full_like(amax, 127.0))
        q = b / scale
        q = (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-128, 127)
    else:
        exp = (torch.frexp(amax).exponent - 9).clamp(-127, 127)
        scale = torch.ldexp(torch.ones_like(amax), exp)
        q = (b / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return (q * scale).reshape(x.shape)


def _route_own(s):
    import nim_lowprec_b200 as L
    r = s["r"]
    L.routeExperts(s["logits"], r["weights"], r["experts"], r["offsets"], r["row_token"],
                   r["places"], renormalize=s["renorm"])
    return r


def _route_plain(s):
    l, k = s["logits"].float(), s["case"]["k"]
    t, e = l.shape
    order = torch.sort(l, dim=-1, descending=True, stable=True)
    top, idx = order.values[:, :k], order.indices[:, :k]
    some = top > -math.inf
    p = torch.exp(top - torch.where(some[:, :1], top[:, :1], torch.zeros_like(top[:, :1])))
    p = torch.where(some, p, torch.zeros_like(p))
    if s["renorm"]:
        total = p.sum(-1, keepdim=True)
    else:
        total = torch.exp(l - top[:, :1]).sum(-1, keepdim=True)
    p = torch.where(some, p / total, torch.zeros_like(p))
    ids = torch.where(some, idx, torch.full_like(idx, e)).reshape(-1)
    by = torch.sort(ids, stable=True)
    places = torch.empty_like(ids)
    places[by.indices] = torch.arange(t * k, device="cuda")
    offsets = torch.searchsorted(by.values, torch.arange(e + 1, device="cuda"))
    return dict(weights=p, experts=torch.where(some, idx, torch.full_like(idx, -1)).int(),
                offsets=offsets.int(),
                row_token=torch.where(by.values < e, by.indices // k,
                                      torch.full_like(by.values, -1)).int(),
                places=torch.where(some, places.reshape(t, k), torch.full_like(idx, -1)).int())


def _decoded(w):
    """Weights in fp32 from their codes and scales, over any leading dimensions."""
    codes, scales = w
    if codes.dtype == torch.uint8:
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device="cuda")
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
        v = v.reshape(*codes.shape[:-1], -1)
        s = scales
    else:
        v = codes.float()
        s = torch.ldexp(torch.ones(scales.shape, device="cuda"), scales.int() - 127)
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(v.shape)


def _values(codes, scales):
    s = torch.ldexp(torch.ones(scales.shape, device="cuda"), scales.int() - 127)
    return (codes.float().reshape(*scales.shape, 32) * s[..., None]).reshape(codes.shape)


def _grouped(x, w, offsets, most):
    """x's rows, in the experts' order, times their experts' weights."""
    rows, experts = x.shape[0], w[0].shape[0]
    r = torch.arange(rows, device="cuda")
    e = torch.searchsorted(offsets[1:].long(), r, right=True).clamp(max=experts - 1)
    if rows < experts:
        return torch.matmul(_decoded((w[0][e], w[1][e])), x[:, :, None])[..., 0]
    at = offsets[:-1].long()[:, None] + torch.arange(most, device="cuda")[None]
    y = torch.bmm(x[at.clamp(max=rows - 1)], _decoded(w).transpose(1, 2))
    return y[e, r - offsets[e].long()]


def _gate(h):
    g, u = h.chunk(2, -1)
    return g / (1.0 + torch.exp(-g)) * u


def _gated_own(s):
    import nim_lowprec_b200 as L
    L.expertGemmGated(s["up"], s["codes"], s["scales"], s["r"]["offsets"], *s["rows"],
                      rowToken=s["r"]["row_token"])
    L.dequantizeRows(*s["rows"], s["vals"])
    return s["vals"]


def _gated_plain(s):
    x = _values(s["codes"], s["scales"])[s["r"]["row_token"].long()]
    h = _gate(_grouped(x, s["up"], s["r"]["offsets"], s["most"]))
    return _quantized(h, "mx8").bfloat16()


def _down_own(s):
    import nim_lowprec_b200 as L
    L.expertGemm(s["down"], s["codes"], s["scales"], s["r"]["offsets"], s["out_rows"])
    L.combineExperts(s["out_rows"], s["r"]["weights"], s["r"]["places"], s["out"])
    return dict(rows=s["out_rows"], out=s["out"])


def _down_plain(s):
    y = _grouped(_values(s["codes"], s["scales"]), s["down"], s["r"]["offsets"], s["most"])
    y = y.to(_DT[s["case"]["y"]])
    return dict(rows=y, out=_combined(y, s["r"]).to(y.dtype))


def _combined(y, r):
    return (y.float()[r["places"].long()] * r["weights"][..., None]).sum(1)


def _linear_own(s):
    import nim_lowprec_b200 as L
    L.quantizeRows(s["x"], *s["rows"])
    L.expertGemm(s["w"], *s["rows"], s["offsets"], s["out"])
    return s["out"]


def _linear_plain(s):
    x = _quantized(s["x"].float(), "mx8")
    return torch.matmul(x, _decoded(s["w"])[0].T).to(s["out"].dtype)


def _layer_own(s):
    import nim_lowprec_b200 as L
    r = s["r"]
    L.addRmsNorm(s["x"], s["res"], s["norm"], s["eps"], total=s["total"], codes=s["rows"][0],
                 scales=s["rows"][1])
    L.routeExperts(s["logits"], r["weights"], r["experts"], r["offsets"], r["row_token"],
                   r["places"], renormalize=s["renorm"])
    L.expertGemmGated(s["up"], *s["rows"], r["offsets"], *s["hidden"], rowToken=r["row_token"])
    L.expertGemm(s["down"], *s["hidden"], r["offsets"], s["out_rows"])
    L.combineExperts(s["out_rows"], r["weights"], r["places"], s["out"], residual=s["total"])
    return dict(total=s["total"], out=s["out"])


def _layer_plain(s):
    total, n = _norm_values(s)
    r = _route_plain(s)
    x = _quantized(n, "mx8")[r["row_token"].long()]
    h = _quantized(_gate(_grouped(x, s["up"], r["offsets"], s["most"])), "mx8")
    y = _grouped(h, s["down"], r["offsets"], s["most"]).bfloat16()
    return dict(total=total, out=(total.float() + _combined(y, r)).bfloat16())


_OPS = {"norm": (_norm_plain, _norm_own), "route": (_route_plain, _route_own),
        "gated": (_gated_plain, _gated_own), "down": (_down_plain, _down_own),
        "linear": (_linear_plain, _linear_own), "layer": (_layer_plain, _layer_own)}


# ------------------------------------------------------------------ what a pass cannot do without

def _used(case):
    """How many experts get a row, on average over the draws of the router: k of them per token, each
    as likely as another."""
    e = case["experts"]
    return e * (1.0 - (1.0 - case["k"] / e) ** case["tokens"])


def _weight_bytes(case, m, k):
    return m * k * ((0.5 if case["w"] == "mx4" else 1.0) + 1 / 32)


def work(case):
    op, t = case["op"], case["tokens"]
    if op == "route":
        e, k = case["experts"], case["k"]
        # logits in; weights, experts, rows and places out
        return dict(bytes=4 * t * e + 16 * t * k + 4 * (e + 1), flops=2 * t * e)
    if op == "norm":
        n, x = t * case["dim"], _SIZE[case["x"]]
        rows = n + (4 * n // case["group"] if case["rows"] == "int8" else n // 32)
        # x and the stream in; the stream, y and the rows out; the rows in again and their values out
        return dict(bytes=4 * n * x + 2 * rows + 2 * n, flops=8 * n)
    dim, inner = case["dim"], case["inner"]
    if op == "linear":
        n = t * dim
        return dict(bytes=_weight_bytes(case, inner, dim) + n * _SIZE[case["x"]]
                    + 2 * (n + n // 32) + t * inner * _SIZE[case["y"]], flops=2 * n * inner)
    k = case["k"]
    rows, used = t * k, _used(case)
    hidden = rows * (inner + inner // 32)
    if op == "gated":
        return dict(bytes=used * _weight_bytes(case, 2 * inner, dim) + t * (dim + dim // 32)
                    + 4 * rows + 2 * hidden + 2 * rows * inner, flops=4 * rows * dim * inner)
    if op == "down":
        return dict(bytes=used * _weight_bytes(case, dim, inner) + hidden + 4 * rows * dim
                    + 8 * rows + 2 * t * dim, flops=2 * rows * dim * inner + 2 * rows * dim)
    # the stream twice in, once out, its rows out and in; the router's; the hidden rows and the
    # experts' rows out and in; the sum
    return dict(bytes=8 * t * dim + 2 * t * (dim + dim // 32) + 4 * t * case["experts"]
                + 24 * rows + used * _weight_bytes(case, 3 * inner, dim) + 2 * hidden
                + 4 * rows * dim, flops=6 * rows * dim * inner)


# ------------------------------------------------------------------ the definition in 64 bits

def _round_mx8(x):
    x = x.reshape(x.shape[0], -1, 32)
    exp = (torch.frexp(x.abs().amax(-1, keepdim=True)).exponent - 9).clamp(-127, 127)
    scale = torch.exp2(exp.double())
    y = (x / scale).clamp(-448.0, 448.0)
    # three bits behind the leading one, and steps of 2^-9 below 2^-6
    step = torch.exp2((torch.frexp(y).exponent - 1).clamp(min=-6).double() - 3.0)
    return (torch.round(y / step) * step * scale).flatten(1)


def _exact_weights(codes, scales):
    if codes.dtype == torch.uint8:
        n = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
        m = n % 8
        v = torch.where(m < 4, m * 0.5, torch.where(m == 7, 6.0, m - 2.0)).double()
        v = torch.where(n >= 8, -v, v)
        s = scales.double()
    else:
        v, s = codes.double(), torch.exp2(scales.double() - 127.0)
    return v * s.repeat_interleave(32, -1)


def _exact_experts(x, w, ids, f):
    """f of each row's products with its expert's weights."""
    out = None
    for e in range(w[0].shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if at.numel():
            y = f(x[at] @ _exact_weights(w[0][e], w[1][e]).T)
            out = torch.zeros(x.shape[0], y.shape[1], dtype=y.dtype, device="cuda") \
                if out is None else out
            out[at] = y
    return out


def _exact_gate(h):
    n = h.shape[1] // 2
    return _round_mx8(h[:, :n] * torch.sigmoid(h[:, :n]) * h[:, n:])


def _exact_choice(logits, k, renorm):
    """(experts, weights) of each token."""
    l = logits.double()
    ids = torch.argsort(-l, dim=-1, stable=True)[:, :k]
    none = torch.isinf(l.gather(1, ids))
    l = torch.where(torch.isinf(l).all(-1, keepdim=True), torch.zeros_like(l), l)
    p = torch.softmax(l, -1).gather(1, ids)
    if renorm:
        p = p / p.sum(-1, keepdim=True)
    return ids.masked_fill(none, -1), p.masked_fill(none, 0.0)


def _exact_norm(s):
    r = (s["x"].double() + s["res"].double()).to(s["x"].dtype)
    d = r.double()
    return r, d / torch.sqrt((d * d).mean(-1, keepdim=True) + s["eps"]) * s["norm"].double()


def exact(case, seed):
    global own
    was, own = own, False  # inputs as they are, with nothing laid out
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "norm":
        r, n = _exact_norm(s)
        if case["rows"] == "mx8":
            return dict(total=r, y=n, vals=_round_mx8(n))
        b = n.reshape(n.shape[0], -1, case["group"])
        scale = b.abs().amax(-1, keepdim=True) / 127.0
        q = b / scale
        return dict(total=r, y=n, vals=(torch.sign(q) * torch.floor(q.abs() + 0.5) * scale).flatten(1))
    if op == "route":
        ids, p = _exact_choice(s["logits"], case["k"], s["renorm"])
        return dict(weights=p, experts=None, offsets=None, row_token=None, places=None)
    if op == "linear":
        return _round_mx8(s["x"].double()) @ _exact_weights(s["w"][0][0], s["w"][1][0]).T
    if op == "layer":
        ids, p = _exact_choice(s["logits"], case["k"], True)
        r, n = _exact_norm(s)
        x = _round_mx8(n).repeat_interleave(case["k"], 0)
        h = _exact_experts(x, s["up"], ids.flatten(), _exact_gate)
        y = _exact_experts(h, s["down"], ids.flatten(), lambda v: v.bfloat16().double())
        y = y.reshape(*ids.shape, -1)
        return dict(total=r, out=r.double() + (y * p[..., None]).sum(1))
    off = s["r"]["offsets"].tolist()
    ids = torch.cat([torch.full((b - a,), e, device="cuda")
                     for e, (a, b) in enumerate(zip(off, off[1:]))])
    x = s["codes"].double() * torch.exp2(s["scales"].double() - 127.0).repeat_interleave(32, -1)
    if op == "gated":
        return _exact_experts(x[s["r"]["row_token"].long()], s["up"], ids, _exact_gate)
    y = _exact_experts(x, s["down"], ids, lambda v: v)
    rounded = y.to(_DT[case["y"]]).double()
    out = rounded[s["r"]["places"].long()] * s["r"]["weights"].double()[..., None]
    return dict(rows=y, out=out.sum(1))
