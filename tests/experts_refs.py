"""Plain forms of 8-bit rows, the router and the experts' products, in 64 bits where they round,
and inputs for their tests."""
import torch

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
#: half a unit in the last place, relative, and the half of the smallest step
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rows8(x, kind="mx8", group=32):
    """(codes, scales) of x by the formulas: scale 2^(floor(log2 amax) - 8), 1 for zeros, in a byte,
    and e4m3 codes; or amax / 127 in fp32 and whole numbers."""
    t, k = x.shape
    b = x.float().reshape(t, k // group, group)
    amax = torch.nan_to_num(b, nan=0.0, posinf=torch.inf, neginf=-torch.inf).abs().amax(-1)
    if kind == "int8":
        s = torch.where(amax == 0, torch.ones_like(amax), amax / torch.full_like(amax, 127.0))
        q = b / s[..., None]
        q = (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-128, 127)
        q = torch.nan_to_num(q, nan=-128.0)  # an infinity over an infinite scale, as in quantizeBatch
        return q.to(torch.int8).reshape(t, k), s
    field = amax.view(torch.int32) >> 23
    code = torch.where(amax == 0, torch.full_like(field, 127), (field - 8).clamp(min=0))
    y = b.double() * torch.exp2(127.0 - code.double())[..., None]
    return e4m3(y).reshape(t, k), code.to(torch.uint8)


def e4m3(y):
    """The code of the nearest e4m3 value, ties to even, at most 448 in magnitude."""
    a = y.abs().clamp(max=448.0)
    step = torch.exp2((torch.frexp(a).exponent - 1).clamp(min=-6).double() - 3.0)
    v = torch.round(a / step) * step
    e = (torch.frexp(v).exponent - 1).clamp(min=-6)
    m = torch.where(v < 2.0 ** -6, v * 2.0 ** 9, v * torch.exp2(3.0 - e.double()) + 8.0 * (e + 6).double())
    c = torch.nan_to_num(m).to(torch.int32) + torch.where(torch.signbit(y), 128, 0)
    return torch.where(torch.isnan(y), 0x7f + (c & 128), c).to(torch.uint8).view(torch.float8_e4m3fn)


def empty_rows8(t, k, kind="mx8", group=32, fill=0):
    if kind == "int8":
        return (torch.full((t, k), fill, dtype=torch.int8, device="cuda"),
                torch.full((t, k // group), float(fill), device="cuda"))
    return (torch.full((t, k), fill, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
            torch.full((t, k // 32), fill, dtype=torch.uint8, device="cuda"))


def values(codes, scales):
    """The values of 8-bit rows in 64 bits."""
    t, k = codes.shape
    if codes.dtype == torch.int8:
        return (codes.double().reshape(t, scales.shape[1], -1) * scales.double()[..., None]).reshape(t, k)
    v = codes.float().double()
    return v * torch.exp2(scales.view(torch.uint8).double() - 127.0).repeat_interleave(32, -1)


def same(a, b):
    """Equal, a NaN to a NaN."""
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def bits(t):
    return t.contiguous().view(torch.uint8)


def weights(g, experts, rows, cols, kind):
    """(codes, scales, values in 64 bits) of experts' weights, with scales over 2^-9 .. 2^2."""
    s = torch.randint(118, 130, (experts, rows, cols // 32), generator=g, device="cuda")
    if kind == "mx4":
        n = torch.randint(0, 16, (experts, rows, cols), generator=g, device="cuda")
        codes = (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8)
        v = E2M1.cuda()[n & 7].double() * torch.where(n >= 8, -1.0, 1.0)
        scales = torch.exp2(s.float() - 127.0)
    else:
        c = torch.randint(0, 256, (experts, rows, cols), generator=g, device="cuda")
        c = torch.where((c & 127) == 127, c - 1, c).to(torch.uint8)  # (no NaN)
        codes = c.view(torch.float8_e4m3fn)
        s = s - 6  # (codes are up to 448)
        v = codes.float().double()
        scales = s.to(torch.uint8)
    return codes, scales, v * torch.exp2(s.double() - 127.0).repeat_interleave(32, -1)


def segments(counts, experts, pad=0):
    """offsets of experts with such numbers of rows."""
    c = torch.tensor(counts[:experts] + [0] * (experts - len(counts)), dtype=torch.int32)
    off = torch.zeros(experts + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(c, 0)
    return off.cuda()


def product(w, x, offsets, rowToken=None):
    """(y, a) in 64 bits: y[r] = W[e] x[t], a[r] = |W[e]| |x[t]|; rows of no expert are NaN."""
    rows = x.shape[0] if rowToken is None else rowToken.numel()
    y = torch.full((rows, w.shape[1]), torch.nan, dtype=torch.float64, device="cuda")
    a = y.clone()
    off = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(off, off[1:])):
        if hi > lo:
            at = torch.arange(lo, hi, device="cuda") if rowToken is None else rowToken[lo:hi].long()
            in_range = (at >= 0) & (at < x.shape[0])
            xe = torch.where(in_range[:, None], x[at.clamp(0, x.shape[0] - 1)], 0.0)
            y[lo:hi] = xe @ w[e].T
            a[lo:hi] = xe.abs() @ w[e].abs().T
    return y, a


def sum_error(cols):
    """What a sum over cols in fp32 may be off, of the sum of magnitudes: every step of 32 products is
    exact up to one cut of a unit in the last place of the running sum, and its own sum up to two."""
    return (cols / 32 + 2) * 2.0 ** -23


def check_product(out, y, a, cols):
    some = ~torch.isnan(y)
    err = (out.double() - y).abs()
    tol = a * sum_error(cols) * (1 + 2.0 ** -7) + y.abs() * HALF_ULP[out.dtype] + TINY[out.dtype]
    bad = some & ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol)[some].max()))


def gate(y, a, cols):
    """(h, e): silu(g) u in 64 bits and what fp32 sums, its fast exponential and quotient may change."""
    g, u = y.chunk(2, -1)
    eg, eu = (t * sum_error(cols) for t in a.chunk(2, -1))
    sig = torch.sigmoid(g)
    h = g * sig * u
    # |silu'| <= 1.1; exp(-g) is off by 2 + 1.2 |g| units of 2^-23, the quotient by 2, two products by 1
    e = 1.1 * eg * u.abs() + (g * sig).abs() * eu + h.abs() * (1.2 * g.abs() + 8.0) * 2.0 ** -23
    return h, e


def check_rows8(codes, scales, h, e):
    """MXFP8 rows of h (rows of no expert NaN), whose elements may be off by e before they round."""
    some = ~torch.isnan(h[:, :1]).expand_as(h)
    hz, ez = torch.nan_to_num(h), torch.nan_to_num(e)
    amax = hz.abs().reshape(h.shape[0], -1, 32).amax(-1).repeat_interleave(32, -1)
    # half a step of three bits, or of the smallest, 2^-10 of a scale that is at most amax 2^-8 (twice
    # that where the largest crosses a power of two); and what is over 448 scales
    low = amax * (1 - 2.0 ** -10)
    most = 448.0 * torch.exp2((torch.frexp(low).exponent - 9).double())
    tol = hz.abs() / 16 + amax * 2.0 ** -17 + (hz.abs() - most).clamp(min=0.0) + ez * 1.07 + 1e-30
    err = (values(codes, scales) - hz).abs()
    bad = some & ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol)[some].max()))


def route(logits, k, renormalize):
    """(experts, weights in 64 bits, offsets, row tokens, places), token by token."""
    l = logits.double().cpu()
    l = torch.where(torch.isnan(l), torch.full_like(l, -torch.inf), l)
    t, n = l.shape
    experts, weight, rows = [], [], [[] for _ in range(n)]
    for i in range(t):
        order = sorted(range(n), key=lambda e: (-l[i, e].item(), e))[:k]
        order = [e if l[i, e] > -torch.inf else -1 for e in order]
        top = l[i].max()
        d = torch.where(l[i] == top, 0.0, l[i] - top) if top > -torch.inf else torch.full((n,), -torch.inf)
        p = torch.exp(d.double())
        some = [e for e in order if e >= 0]
        total = (p[some].sum() if renormalize else p.sum()).item() if some else 1.0
        experts.append(order)
        weight.append([p[e].item() / total if e >= 0 else 0.0 for e in order])
        for j, e in enumerate(order):
            if e >= 0:
                rows[e].append((i, j))
    offsets, token, places = [0], [], [[-1] * k for _ in range(t)]
    for e in range(n):
        for i, j in rows[e]:
            places[i][j] = len(token)
            token.append(i)
        offsets.append(len(token))
    return experts, weight, offsets, token, places
