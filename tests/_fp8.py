"""Plain forms of the e4m3 operators and the router, in fp64 with a bound for each output.

Codes and scales of activations are fixed bit for bit; sums are not, since their order is
the kernel's: bounds count a rounding of 2^-24 of the sum of magnitudes for each term of a block's
sum of 128, or for each group of 8 that the matrix instruction adds up exactly (+ 8 for scalings), and one for each block."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # of the value: half a unit of the last bit
FLOOR = 448.0 * 2.0 ** -126


def nearest(v):
    """fp64 -> the nearest e4m3 value, halves to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def blocks(x):
    """(rows, K) -> (rows, K / 128, 128), zeros behind the end."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % 128)).unflatten(-1, (-1, 128))


def quant(x):
    """(codes as fp64 values (rows, K), scales fp64 (rows, K / 128)) of x (rows, K) of any type."""
    b = blocks(x.double())
    amax = b.abs().amax(-1).clamp_min(FLOOR)
    q = nearest(b * 448 / amax[..., None])
    bad = ~torch.isfinite(b).all(-1)
    q = torch.where(bad[..., None], 0.0, q)
    s = torch.where(bad, math.nan, amax / 448).float().double()    # the scale is rounded to fp32
    return q.flatten(-2)[..., :x.shape[-1]], s


def spread(s, N, K):
    """Block scales (N / 128, K / 128) -> (N, K)."""
    return s.double().repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]


def exponent(v):
    """Of e4m3 values, in fp64: that of the smallest normal for those below."""
    return torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent.double() - 1


def matrix_sums(q, w):
    """Sums over K of q (M, K) w (N, K), codes in fp64, as the matrix instruction makes them, block by block of 128:
    (M, N, K / 128).  Products of eight neighbours are cut, towards zero, at 2^-13 of the largest sum of
    their operands' exponents; what is left is added up."""
    K = q.shape[1]
    q, w = (torch.nn.functional.pad(t, (0, -K % 128)).unflatten(-1, (-1, 8)) for t in (q, w))
    eq, ew = exponent(q), exponent(w)
    out = torch.empty(q.shape[0], w.shape[0], q.shape[1] // 16, dtype=torch.float64, device=q.device)
    rows = max(1, (1 << 26) // w.numel())
    for r in range(0, q.shape[0], rows):
        p = q[r:r + rows, None] * w
        e = torch.where(p == 0, -100.0, eq[r:r + rows, None] + ew).amax(-1, keepdim=True)
        unit = torch.exp2(e - 13)
        out[r:r + rows] = (torch.trunc(p / unit) * unit).sum(-1).unflatten(-1, (-1, 16)).sum(-1)
    return out


def product(q, s, w, ws, matrix=False):
    """Codes q (M, K) fp64 with scales s (M, K / 128), weights as codes and scales: (y, bound of its error before
    rounding), the products exact or (matrix) as the matrix instruction makes them."""
    N, K = w.shape
    x = q * s.repeat_interleave(128, 1)[:, :K]
    v = w.float().double() * spread(ws, N, K)
    size = x.abs() @ v.abs().t()
    if matrix:
        scale = s[:, None, :] * ws.double().repeat_interleave(128, 0)[:N]
        y = torch.where(scale == 0, 0.0, matrix_sums(q, w.float().double()) * scale).sum(-1)
    else:
        y = x @ v.t()
    return y, ((24 if matrix else 136) + -(-K // 128)) * 2.0 ** -24 * size


def off(y, ref, err, dtype):
    """Largest |y - ref| over its bound; NaN has to meet NaN."""
    y = y.double()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(y), nan)
    bound = UNIT[dtype] * ref.abs() + 1.01 * err + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133)
    ratio = ((y - ref).abs() / bound)[~nan]
    return float(ratio.max()) if ratio.numel() else 0.0


def weights(g, *shape, dev="cpu"):
    """Codes over all of e4m3's range and scales of different size."""
    lead, (N, K) = shape[:-2], shape[-2:]
    w = (torch.randn(*lead, N, K, generator=g) * torch.exp(torch.randn(*lead, N, 1, generator=g))).clamp(-3, 3) * 149
    s = torch.exp(0.5 * torch.randn(*lead, -(-N // 128), -(-K // 128), generator=g)) * 2.0 ** -12
    return w.to(E4M3).to(dev), s.to(dev)


def route(x, k, bias=None, sigmoid=False, groups=1, keep=1, best=1, renorm=True, scale=1.0):
    """Row by row in Python's terms: (weights fp64, ids)."""
    x = x.double().cpu()
    T, E = x.shape
    if sigmoid:
        s = 1 / (1 + torch.exp(-x))
    else:
        s = torch.softmax(x, -1)
        s = torch.where((x == -math.inf).all(-1, keepdim=True), 0.0, s)
    c = s if bias is None else s + bias.double().cpu()
    ids = torch.empty(T, k, dtype=torch.int64)
    low = -math.inf

    def order(v):                                                   # NaN below every number
        return (0, 0.0) if v != v else (1, v)

    for t in range(T):
        allowed = range(E)
        if groups > 1:
            size = E // groups
            score = []
            for g in range(groups):
                top = sorted((float(v) for v in c[t, g * size:(g + 1) * size]), key=order, reverse=True)[:best]
                score.append(sum(top))
            kept = sorted(range(groups), key=lambda g: (order(score[g]), -g), reverse=True)[:keep]
            allowed = [e for g in kept for e in range(g * size, (g + 1) * size)]
        ids[t] = torch.tensor(sorted(allowed, key=lambda e: (order(float(c[t, e])), -e), reverse=True)[:k])
    w = s.gather(1, ids)
    if renorm:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return w * scale, ids


def experts(x, wts, ids, w_up, s_up, w_down, s_down, up_matrix, down_matrix, rows=0.0):
    """(y, bound of its error before rounding).  The hidden values' codes may fall to either side of a half where the
    kernel's sums leave that open: such a code counts a whole step, and its row's cut products whatever they may (7 of 8
    products, each by less than 2^-13 of the group's largest).  up_matrix, down_matrix: which products are cut; rows:
    half a unit, of the value, of the type that experts' rows are kept in."""
    E, N2, H = w_up.shape
    I = N2 // 2
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(y)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        a, ea = product(*quant(x[t]), w_up[e], s_up[e], up_matrix)
        g, u, eg, eu = a[:, :I], a[:, I:], ea[:, :I], ea[:, I:]
        h = g * torch.sigmoid(g) * u
        eh = 1.1 * u.abs() * eg + (g * torch.sigmoid(g)).abs() * eu + 1.1 * eg * eu + 2.0 ** -21 * h.abs()
        b, eb = blocks(h), blocks(eh)
        amax = b.abs().amax(-1, keepdim=True).clamp_min(FLOOR)
        ea_max = eb.amax(-1, keepdim=True)
        v = b * 448 / amax
        ev = 448 * (eb / amax + b.abs() * ea_max / amax ** 2) + v.abs() * 2.0 ** -22
        lo, hi = nearest(v - ev), nearest(v + ev)
        s = amax / 448
        code = nearest(v)
        step = torch.maximum((hi - code).abs(), (code - lo).abs())
        dh = (step * s + code.abs() * s * (ea_max / amax + 2.0 ** -22)).flatten(-2)
        o, eo = product(code.flatten(-2), s[..., 0], w_down[e], s_down[e], down_matrix)
        hv = (code * s).flatten(-2).abs()
        wd = (w_down[e].float().double() * spread(s_down[e], H, I)).abs()
        eo = eo + dh @ wd.t()
        if down_matrix:
            eo = eo + (step.amax((1, 2)) > 0)[:, None] * 7 * 2.0 ** -13 * (hv @ wd.t())
        w = wts[t, j].double()[:, None]
        y.index_add_(0, t, o * w)
        err.index_add_(0, t, (eo + (2.0 ** -22 + rows) * o.abs()) * w.abs())
    return y, err
