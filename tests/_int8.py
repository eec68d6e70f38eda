"""Plain forms of the 8-bit operators on the CPU.

What is fixed bit for bit (codes, scales, rotations, the integer product and
its scaling) is computed in fp32 with the formulas' own steps; attention in
fp64 with a bound for each output."""
from __future__ import annotations

import math

import torch

TINY, FLOOR = 2.0 ** -126, 2.0 ** -40
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # rounding to 8 and 11 significant bits: half a unit of the last


def quant_token(x):
    xf = x.float()
    amax = xf.abs().amax(-1)
    s = (amax / 127).clamp_min(TINY)
    q = (xf * (1.0 / s)[..., None]).round().clamp(-127, 127)
    bad = ~torch.isfinite(xf).all(-1)
    return torch.where(bad[..., None], torch.zeros_like(q), q).to(torch.int8), torch.where(bad, torch.full_like(s, math.nan), s)


def product(xq, xs, wq, ws, dtype):
    """The exact integer sum (in fp64: below 2^53), then the two fp32 products."""
    acc = xq.reshape(-1, xq.shape[-1]).double() @ wq.double().t()
    y = acc.float() * xs.reshape(-1, 1) * ws
    return y.to(dtype).reshape(*xq.shape[:-1], wq.shape[0])


def table_of(positions, rot, theta=10000.0):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    return torch.cat((a.cos(), a.sin()), 1).float()


def rotate(x, pos, cos_sin, interleaved):
    """x (tokens, heads, D) in fp32."""
    x = x.float().clone()
    rot = cos_sin.shape[1]
    cs = cos_sin[pos.clamp(0, cos_sin.shape[0] - 1)][:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + (1 if interleaved else rot // 2)
    a, b = x[..., ia], x[..., ib]
    x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
    return x


class Cache:
    """pages of codes and scales on the CPU; values as (pages, heads, D, page)."""

    def __init__(self, pages, heads, page, D, fill=0, scale=math.nan):
        self.k = torch.full((pages, heads, page, D), fill, dtype=torch.int8)
        self.v = torch.full((pages, heads, D, page), fill, dtype=torch.int8)
        self.ks = torch.full((pages, heads), scale)
        self.vs = torch.full((pages, heads), scale)
        self.page, self.D, self.heads = page, D, heads

    def tensors(self):
        return self.k, self.v, self.ks, self.vs

    def to(self, dev):
        return [t.to(dev) for t in self.tensors()]

    def append(self, seq_pages, start, k, v):
        """k, v (n, heads, D) fp32, already rotated, at positions start on."""
        n, at = k.shape[0], 0
        while at < n:
            p, o = divmod(start + at, self.page)
            m = min(self.page - o, n - at)
            if p < len(seq_pages) and 0 <= seq_pages[p] < self.k.shape[0]:
                self._put(self.k, self.ks, seq_pages[p], o, k[at:at + m], False)
                self._put(self.v, self.vs, seq_pages[p], o, v[at:at + m], True)
            at += m

    def _put(self, codes, scales, page, o, x, values):
        for h in range(self.heads):
            tile = codes[page, h].t() if values else codes[page, h]          # (page, D)
            new = x[:, h]
            old = scales[page, h] if o else torch.tensor(0.0)
            fin = bool(torch.isfinite(new).all()) and not bool(torch.isnan(old))
            if not fin:
                scales[page, h] = math.nan
                tile[o:o + new.shape[0]] = 0
                continue
            s = torch.maximum(old, (new.abs().amax() / 127).clamp_min(FLOOR))
            if o and s != old:
                tile[:o] = (tile[:o].float() * (old / s)).round().to(torch.int8)
            tile[o:o + new.shape[0]] = (new * (1.0 / s)).round().clamp(-127, 127).to(torch.int8)
            scales[page, h] = s

    def sequence(self, seq_pages, length):
        """(k, v) of the first `length` tokens, (length, heads, D) fp64, and which of them a page holds."""
        k = torch.zeros(length, self.heads, self.D, dtype=torch.float64)
        v, seen = k.clone(), torch.zeros(length, dtype=torch.bool)
        for p in range(-(-length // self.page)):
            lo, hi = p * self.page, min(length, (p + 1) * self.page)
            if p < len(seq_pages) and 0 <= seq_pages[p] < self.k.shape[0]:
                i = seq_pages[p]
                k[lo:hi] = (self.k[i].double() * self.ks[i].double()[:, None, None]).transpose(0, 1)[:hi - lo]
                v[lo:hi] = (self.v[i].double() * self.vs[i].double()[:, None, None]).permute(2, 0, 1)[:hi - lo]
                seen[lo:hi] = True
        return k, v, seen


def attention(q, k, v, seen, first, scale, window=0, cap=0.0):
    """q (n, Hq, D) at positions first on; k, v (L, Hkv, D) fp64.  (out, A, E)
    in fp64: the outputs, the sums of p |v| and a bound of the error of the scores
    (in natural units) that fp32 sums of exact products of D terms have.  Where that is
    1/16 or more, A is made so that the bound says what is left: outputs lie among the values."""
    n, Hq, D = q.shape
    L, H = k.shape[:2]
    q = q.double()
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    A, E = out.clone(), torch.zeros(n, Hq, 1, dtype=torch.float64)
    if L == 0:
        return out, A, E
    pos = first + torch.arange(n)[:, None]
    t = torch.arange(L)
    ok = (t <= pos) & seen
    if window:
        ok &= t > pos - window
    for hq in range(Hq):
        kk, vv = k[:, hq // (Hq // H)], v[:, hq // (Hq // H)]
        s = q[:, hq] @ kk.t() * scale
        size = (q[:, hq].abs() @ kk.abs().t() * abs(scale)).masked_fill(~ok, 0.0)
        if cap:
            s = cap * torch.tanh(s / cap)
        s = s.masked_fill(~ok, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
        p = torch.where(ok, p / p.sum(-1, keepdim=True).clamp_min(1e-300), 0.0)
        out[:, hq] = p @ torch.nan_to_num(vv) if not torch.isnan(s[ok]).any() else torch.where(ok, p, 0.0) @ vv
        A[:, hq] = p @ torch.nan_to_num(vv).abs()
        # products of a code and q's 8 or 11 bits are exact; D rounded additions
        # and the scalings; the exponent's argument, itself rounded a few times
        top = s.masked_fill(~ok, 0.0).abs().amax(-1, keepdim=True)
        e = (D + 8) * 2.0 ** -24 * size.amax(-1, keepdim=True) + 2.0 ** -21 * (top + cap + 64)
        lost = e >= 1 / 16                                  # first-order bounds do not hold
        most = torch.where(ok[..., None], torch.nan_to_num(vv).abs()[None], 0.0).amax(1)
        E[:, hq] = torch.where(lost, 1.0, e)
        A[:, hq] = torch.where(lost, most, A[:, hq])
    return out, A, E


def attention_bound(out, A, E, dtype):
    """|kernel - out| of a correct kernel is below this: output rounding; each weight
    rounded to fp16 (2^-11) and off by twice the scores' error, above and below
    the fraction; the smallest weights fall short by at most 2^-26 of the largest."""
    return UNIT[dtype] * out.abs() * 1.01 + (2.0 ** -11 + 2.0 ** -20 + 2.02 * E) * A * 1.01 + 2.0 ** -25
