"""The 8-bit operators around the W4A4 layers, as measured cases.

A decoder layer whose feed-forward part runs in W4A4 needs, beside it:

* ``linear``: a projection in 8-bit integers, activations scaled per token and
  weights per output channel (query/key/value and output projections, and the
  feed-forward layers that 4 bits are too few for);
* ``append``: one step's keys and values rotated by position and written into
  a paged 8-bit cache with a scale for each page and head, the queries rotated
  on the way; the pages it touched are read back as values;
* ``decode``: attention of one new token per sequence over that cache;
* ``chunk``: the same for many new tokens per sequence (prefill, or a chunk of
  it behind an earlier context), causal, optionally with a sliding window and
  scores capped by a tanh.

The cache holds pages of ``page`` tokens: keys (pages, heads, page, D), values
(pages, heads, D, page), int8, and fp32 scales (pages, heads) of each.  A page's
scale is its largest magnitude / 127 and grows with it: the codes that are
there already are then rescaled.  ``block_table`` lists each sequence's pages.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TINY = 2.0 ** -126                     # smallest scale of an activation row
FLOOR = 2.0 ** -40                     # smallest scale of a cache page
LARGEST = 4096 * 57344 * 8192          # M * N * K of the largest linear case
TOKENS = 2 ** 28                       # sequences * length * Hkv * D of the largest cache
SCORES = 2 ** 31                       # sequences * Hq * new tokens * length of the largest chunk


def listed():
    return [
        # one token of one user, a small square projection: launches and latency
        {"name": "linear 1x4096x4096", "kind": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # one token through a 70B feed-forward layer held in 8 bits: the weight stream
        {"name": "linear 1x57344x8192", "kind": "linear", "M": 1, "N": 57344, "K": 8192, "dtype": "bf16"},
        # a ragged small batch
        {"name": "linear 13x24576x4096", "kind": "linear", "M": 13, "N": 24576, "K": 4096, "dtype": "fp16"},
        # a short prompt of odd length, square projection
        {"name": "linear 203x8192x8192", "kind": "linear", "M": 203, "N": 8192, "K": 8192, "dtype": "bf16"},
        # the largest: long-prompt prefill of a 70B feed-forward layer
        {"name": "linear 4096x57344x8192", "kind": "linear", "M": 4096, "N": 57344, "K": 8192, "dtype": "bf16"},
        # a decode step of 64 users: one token each, behind ragged contexts
        {"name": "append 64x1", "kind": "append", "dtype": "bf16", "B": 64, "n": 1, "L": 4096, "Hq": 64, "Hkv": 8,
         "D": 128, "page": 64, "rot": 128, "interleaved": False},
        # three ragged prompts, the first of them behind a context
        {"name": "append 3x2000", "kind": "append", "dtype": "bf16", "B": 3, "n": 2000, "L": 2500, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "rot": 128, "interleaved": False},
        # three users in the middle of short answers, a head for each query, small heads
        {"name": "decode 3x300", "kind": "decode", "dtype": "fp16", "B": 3, "n": 1, "L": 300, "Hq": 32, "Hkv": 32,
         "D": 64, "page": 16, "window": 0, "cap": 0.0},
        # one user with a long document: the cache's stream has to be split
        {"name": "decode 1x131072", "kind": "decode", "dtype": "bf16", "B": 1, "n": 1, "L": 131072, "Hq": 64, "Hkv": 8,
         "D": 128, "page": 64, "window": 0, "cap": 0.0},
        # continuous batching with ragged lengths
        {"name": "decode 64x4096", "kind": "decode", "dtype": "bf16", "B": 64, "n": 1, "L": 4096, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "window": 0, "cap": 0.0},
        # a long prompt
        {"name": "chunk 1x8192", "kind": "chunk", "dtype": "bf16", "B": 1, "n": 8192, "L": 8192, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "window": 0, "cap": 0.0},
        # ragged chunks behind contexts, in layers with a sliding window and capped scores
        {"name": "chunk 5x700+", "kind": "chunk", "dtype": "fp16", "B": 5, "n": 700, "L": 3700, "Hq": 16, "Hkv": 4,
         "D": 64, "page": 32, "window": 1024, "cap": 30.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of those ranges: every number of rows or new tokens up to
    the largest, odd widths and lengths, several head layouts and pages."""
    kind = rng.choice(["linear"] * 3 + ["append"] * 2 + ["decode"] * 3 + ["chunk"] * 2)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "linear":
        step = 64 if rng.random() < 0.25 else 256
        K = max(step, _log(rng, 1024, 16384) // step * step)
        N = _log(rng, 512, 57344)
        if rng.random() < 0.7:
            N = (N + 63) // 64 * 64
        N = min(N, 57344 * 8192 // K)
        return {"kind": kind, "M": min(_log(rng, 1, 4096), LARGEST // (N * K)), "N": N, "K": K, "dtype": dtype}
    Hq, Hkv = rng.choice([(32, 8), (64, 8), (32, 32), (16, 1), (40, 8), (28, 4)])
    D = rng.choice([64, 128, 128])
    case = {"kind": kind, "dtype": dtype, "Hq": Hq, "Hkv": Hkv, "D": D, "page": rng.choice([16, 32, 64, 128])}
    if kind == "append":
        if rng.random() < 0.5:
            B, n, L = _log(rng, 1, 128), 1, _log(rng, 1, 8192)
        else:
            B, n = rng.randint(1, 6), _log(rng, 2, 2048)
            L = n + rng.choice([0, _log(rng, 1, 4096)])
        return {**case, "B": B, "n": n, "L": min(L, TOKENS // (B * Hkv * D)),
                "rot": rng.choice([D, D, D // 2]), "interleaved": rng.random() < 0.25}
    if kind == "decode":
        B, n = _log(rng, 1, 64), 1
        L = _log(rng, 1, min(131072, TOKENS // (B * Hkv * D)))
    else:
        B, n = rng.randint(1, 6), _log(rng, 2, 4096)
        n = min(n, math.isqrt(SCORES // (B * Hq)))
        L = n + min(rng.choice([0, _log(rng, 1, 8192)]), SCORES // (B * Hq * n) - n)
        L = max(n, min(L, TOKENS // (B * Hkv * D)))
    window = _log(rng, 16, 4096) if rng.random() < 0.25 else 0
    return {**case, "B": B, "n": n, "L": L, "window": window, "cap": rng.choice([0.0, 0.0, 0.0, 30.0])}


# ------------------------------------------------------------------- inputs
def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _lengths(case):
    """(new tokens, total length) of each sequence, ragged, the first the longest."""
    n = [max(1, case["n"] - b * 613 % (case["n"] * 3 // 4 + 1)) for b in range(case["B"])]
    room = case["L"] - case["n"]
    return n, [n[b] + room - b * 7919 % (room * 3 // 4 + 1) for b in range(case["B"])]


def _linear_inputs(case, seed):
    g = _generator(seed, 11)
    M, N, K = case["M"], case["N"], case["K"]
    x = torch.randn(M, K, generator=g, device=DEV)
    x[:, torch.randperm(K, generator=g, device=DEV)[: K // 100]] *= 20.0     # outlier channels
    w = torch.empty(N, K, dtype=torch.int8, device=DEV)
    for r in range(0, N, 8192):
        w[r:r + 8192] = torch.randn(min(8192, N - r), K, generator=g, device=DEV).mul_(30).round_().clamp_(-127, 127)
    ws = torch.exp(0.2 * torch.randn(N, generator=g, device=DEV)) * (0.02 / 30)
    return x.to(DTYPES[case["dtype"]]), w, ws


def _cache(case, filled, g):
    """Pages in a random order with the first `filled` tokens of each sequence
    in them, N(0, 1) by channels of different size."""
    B, Hkv, D, ps = case["B"], case["Hkv"], case["D"], case["page"]
    lens = _lengths(case)[1]
    per = [-(-n // ps) for n in lens]
    total = sum(per)
    ids = torch.randperm(total + 3, generator=g, device=DEV)[:total].to(torch.int32)
    table = torch.full((B, max(per)), -1, dtype=torch.int32, device=DEV)
    left = torch.zeros(total, dtype=torch.int64, device=DEV)     # filled tokens from a page's start on
    at = 0
    for b in range(B):
        table[b, :per[b]] = ids[at:at + per[b]]
        left[at:at + per[b]] = filled[b] - ps * torch.arange(per[b], device=DEV)
        at += per[b]
    here = torch.arange(ps, device=DEV) < left[:, None]          # (pages, page)
    out = []
    for _ in range(2):
        codes = torch.zeros(total + 3, Hkv, ps, D, dtype=torch.int8, device=DEV)
        scale = torch.full((total + 3, Hkv), FLOOR, device=DEV)
        size = torch.exp(0.4 * torch.randn(Hkv, 1, D, generator=g, device=DEV))
        for p in range(0, total, 2048):
            x = torch.randn(min(2048, total - p), Hkv, ps, D, generator=g, device=DEV)
            x = x * size * here[p:p + 2048, None, :, None]
            s = (x.abs().amax((2, 3)) / 127).clamp_min(FLOOR)
            codes[ids[p:p + 2048].long()] = (x / s[..., None, None]).round().to(torch.int8)
            scale[ids[p:p + 2048].long()] = s
        out.append((codes, scale))
    (kc, ks), (vc, vs) = out
    return kc, vc.transpose(2, 3).contiguous(), ks, vs, table


def _starts(n):
    cu = [0]
    for v in n:
        cu.append(cu[-1] + v)
    return cu


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _append_inputs(case, seed):
    g = _generator(seed, 23)
    n, lens = _lengths(case)
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    cache = _cache(case, [m - k for m, k in zip(lens, n)], g)
    T = sum(n)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=DEV).to(DTYPES[case["dtype"]])
    freq = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
    angle = torch.arange(max(lens), dtype=torch.float64, device=DEV)[:, None] * freq
    # the pages that the step touches, which its program knows
    rows = [(b, p) for b in range(case["B"]) for p in range((lens[b] - n[b]) // ps, (lens[b] - 1) // ps + 1)]
    where = torch.tensor(rows, device=DEV)
    return {"q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hkv], "v": qkv[:, Hq + Hkv:],
            "cos_sin": torch.cat((angle.cos(), angle.sin()), 1).float(), "cache": cache[:4], "table": cache[4],
            "lens": _int32(lens), "cu": _int32(_starts(n)) if case["n"] > 1 else None, "where": where,
            "pages": cache[4][where[:, 0], where[:, 1]].contiguous()}


def _attention_inputs(case, seed):
    g = _generator(seed, 29)
    n, lens = _lengths(case)
    cache = _cache(case, lens, g)
    q = torch.randn(sum(n), case["Hq"], case["D"], generator=g, device=DEV) * 1.5
    return {"q": q.to(DTYPES[case["dtype"]]), "cache": cache[:4], "table": cache[4], "lens": _int32(lens),
            "cu": _int32(_starts(n)) if case["kind"] == "chunk" else None, "most": max(n), "max_len": max(lens)}


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "linear":
        state["args"] = _linear_inputs(case, seed)
    else:
        state.update(_append_inputs(case, seed) if case["kind"] == "append" else _attention_inputs(case, seed))
    return state


# -------------------------------------------------- the operators in plain form
def _plain_linear(x, w, ws):
    xf = x.float()
    s = (xf.abs().amax(-1, keepdim=True) / 127).clamp_min(TINY)
    q = (xf * (1.0 / s)).round().clamp(-127, 127)
    return ((q @ w.float().t()) * s * ws).to(x.dtype)


def _plain_rotate(x, c, s, interleaved):
    x = x.float()
    rot = 2 * c.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * s, b * c + a * s
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_page(codes, scale, new, is_new, is_old):
    """One tensor's touched pages, (pages, heads, page, D), after the append."""
    x = torch.where(is_new, new, 0.0)
    old = torch.where(is_old.any(2, keepdim=True), scale[..., None, None], 0.0)
    s = torch.maximum(old, (x.abs().amax((2, 3), keepdim=True) / 127).clamp_min(FLOOR))
    kept = torch.where(is_old, (codes.float() * (old / s)).round(), codes.float())
    return torch.where(is_new, (x * (1.0 / s)).round().clamp(-127, 127), kept), s


def _plain_append(st):
    kc, vc, ks, vs = st["cache"]
    case, table, lens, where, pages = st["case"], st["table"], st["lens"].long(), st["where"], st["pages"].long()
    B, T, ps, D = case["B"], st["q"].shape[0], case["page"], case["D"]
    cu = torch.arange(B + 1, device=DEV) if st["cu"] is None else st["cu"].long()
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, t, right=True) - 1
    start = lens - cu.diff()
    pos = start[seq] + t - cu[seq]
    c, s = st["cos_sin"][pos][:, None].chunk(2, -1)
    q = _plain_rotate(st["q"], c, s, case["interleaved"]).to(st["q"].dtype)
    k, v = _plain_rotate(st["k"], c, s, case["interleaved"]), st["v"].float()
    b = where[:, :1]
    pos = where[:, 1:] * ps + torch.arange(ps, device=DEV)               # (touched pages, page)
    is_new = ((pos >= start[b]) & (pos < lens[b]))[:, None, :, None]
    is_old = (pos < start[b])[:, None, :, None]
    token = (cu[b] + pos - start[b]).clamp(0, T - 1)
    kq, kscale = _plain_page(kc[pages], ks[pages], k[token].transpose(1, 2), is_new, is_old)
    vq, vscale = _plain_page(vc[pages].transpose(2, 3), vs[pages], v[token].transpose(1, 2), is_new, is_old)
    kc[pages], vc[pages] = kq.to(torch.int8), vq.to(torch.int8).transpose(2, 3)
    ks[pages], vs[pages] = kscale[..., 0, 0], vscale[..., 0, 0]
    return {"q": q, "k": (kq * kscale).to(q.dtype), "v": (vq * vscale).to(q.dtype)}


def _plain_attention(st):
    kc, vc, ks, vs = st["cache"]
    case, q, lens = st["case"], st["q"], st["lens"].long()
    B, Hkv, D, most = case["B"], case["Hkv"], case["D"], st["most"]
    G, T = case["Hq"] // Hkv, q.shape[0]
    table = st["table"].long().clamp_min(0)
    k = kc[table].float() * ks[table][..., None, None]                   # (B, pages, Hkv, page, D)
    v = vc[table].float() * vs[table][..., None, None]
    k = k.transpose(1, 2).reshape(B, Hkv, -1, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hkv, -1, D)
    cu = torch.arange(B + 1, device=DEV) if st["cu"] is None else st["cu"].long()
    i = torch.arange(most, device=DEV)
    rows = q.float()[(cu[:-1, None] + i).clamp_max(T - 1)]               # (B, most, Hq, D)
    rows = rows.view(B, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * most, D)
    s = (rows @ k.transpose(2, 3)).view(B, Hkv, G, most, -1) * D ** -0.5
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    at = (lens - cu.diff())[:, None, None] + i[:, None]                  # (B, most, 1): a row's position
    col = torch.arange(s.shape[-1], device=DEV)
    seen = (col <= at) & (col < lens[:, None, None])
    if case["window"]:
        seen &= col > at - case["window"]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.reshape(B, Hkv, G * most, -1) @ v).view(B, Hkv, G, most, D)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o.permute(0, 3, 1, 2, 4)[b, t - cu[b]].reshape(T, -1, D).to(q.dtype)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        if kind == "linear":
            return _plain_linear(*state["args"])
        return _plain_append(state) if kind == "append" else _plain_attention(state)
    from my_int4 import _C
    if kind == "linear":
        return _C.w8a8_linear(*state["args"])
    if kind == "append":
        q = _C.kv8_append(state["q"], state["k"], state["v"], state["cos_sin"], *state["cache"], state["table"],
                          state["lens"], cu_q=state["cu"], interleaved=state["case"]["interleaved"])
        k, v = _C.kv8_read(*state["cache"], state["pages"], q.dtype)
        return {"q": q, "k": k, "v": v}
    return _C.kv8_attention(state["q"], *state["cache"], state["table"], state["lens"], cu_q=state["cu"],
                            window=state["case"]["window"], softcap=state["case"]["cap"], max_len=state["max_len"])


def _seen(case):
    """Pairs of a query and a token that it sees, over the sequences."""
    pairs = 0
    for n, m in zip(*_lengths(case)):
        for at in (range(m - n, m) if case["window"] else ()):
            pairs += min(at + 1, case["window"])
        if not case["window"]:
            pairs += n * (m - n) + n * (n + 1) // 2
    return pairs


def work(case):
    """Bytes: inputs read once, outputs written once; operations: the products."""
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * M * K + N * K + 4 * N + 2 * M * N, "flops": 2 * M * N * K}
    n, lens = _lengths(case)
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    T = sum(n)
    if case["kind"] == "append":
        pages = sum((m - 1) // ps - (m - k) // ps + 1 for k, m in zip(n, lens))
        read_back = pages * Hkv * ps * D * 2 * (1 + 2)
        return {"bytes": 2 * T * D * (2 * Hq + 2 * Hkv) + 4 * T * case["rot"] + 2 * T * Hkv * D + read_back,
                "flops": 3 * T * case["rot"] * (Hq + Hkv)}
    tokens = sum(min(m, case["window"] + k - 1) if case["window"] else m for k, m in zip(n, lens))
    return {"bytes": 2 * tokens * Hkv * D + 4 * T * Hq * D, "flops": 4 * _seen(case) * Hq * D}


# ------------------------------------------------------------ in 64 bits
def _exact_linear(x, w, ws):
    x = x.double()
    s = x.abs().amax(-1, keepdim=True) / 127
    q = torch.round(x / s)
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    for r in range(0, w.shape[0], 8192):
        y[:, r:r + 8192] = q @ w[r:r + 8192].double().t().contiguous()
    return y * s * ws.double()


def _exact_append(case, st):
    """Sequence by sequence and page by page; rotations as complex products."""
    n, lens = _lengths(case)
    ps, half = case["page"], case["rot"] // 2

    def turn(x, lo, hi):
        z = torch.complex(*(t[:, None].double() for t in st["cos_sin"][lo:hi].split(half, 1)))
        x = x.double().clone()
        r = x[..., :2 * half]
        re, im = (r[..., ::2], r[..., 1::2]) if case["interleaved"] else (r[..., :half], r[..., half:])
        w = torch.complex(re.contiguous(), im.contiguous()) * z
        re.copy_(w.real)
        im.copy_(w.imag)
        return x

    kc, vc, ks, vs = (t.double() for t in (a[st["pages"].long()] for a in st["cache"]))
    out = {"q": [], "k": [], "v": []}
    at = row = 0
    for b in range(case["B"]):
        lo, hi = lens[b] - n[b], lens[b]
        out["q"].append(turn(st["q"][at:at + n[b]], lo, hi))
        new = {"k": turn(st["k"][at:at + n[b]], lo, hi), "v": st["v"][at:at + n[b]].double()}
        at += n[b]
        for p in range(lo // ps, (hi - 1) // ps + 1):
            f, e = max(lo, p * ps), min(hi, (p + 1) * ps)
            for name, codes, scale in (("k", kc[row], ks[row]), ("v", vc[row].transpose(1, 2), vs[row])):
                x = new[name][f - lo:e - lo].transpose(0, 1)                 # (heads, tokens, D)
                s = (x.abs().amax((1, 2)) / 127).clamp_min(FLOOR)
                if f > p * ps:
                    s = torch.maximum(s, scale)
                s = s[:, None, None]
                y = torch.zeros_like(codes)
                y[:, :f - p * ps] = torch.round(codes[:, :f - p * ps] * scale[:, None, None] / s) * s
                y[:, f - p * ps:e - p * ps] = torch.round(x / s) * s
                out[name].append(y)
            row += 1
    return {"q": torch.cat(out["q"]), "k": torch.stack(out["k"]), "v": torch.stack(out["v"])}


def _exact_attention(case, st):
    """Sequence by sequence and head by head."""
    kc, vc, ks, vs = st["cache"]
    n, lens = _lengths(case)
    G, D = case["Hq"] // case["Hkv"], case["D"]
    out = torch.zeros(sum(n), case["Hq"], D, dtype=torch.float64, device=DEV)
    first = 0
    for b in range(case["B"]):
        pages = st["table"][b, :-(-lens[b] // case["page"])].long()
        j = torch.arange(lens[b], device=DEV)
        i = torch.arange(lens[b] - n[b], lens[b], device=DEV)[:, None]
        hidden = j > i
        if case["window"]:
            hidden |= j <= i - case["window"]
        for h in range(case["Hkv"]):
            k = (kc[pages, h].double() * ks[pages, h].double()[:, None, None]).reshape(-1, D)[:lens[b]]
            v = (vc[pages, h].double() * vs[pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)[:lens[b]]
            for r in range(h * G, h * G + G):
                s = (st["q"][first:first + n[b], r].double() @ k.t().contiguous()) / math.sqrt(D)
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                out[first:first + n[b], r] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v
        first += n[b]
    return out


def exact(case, seed):
    if case["kind"] == "linear":
        return _exact_linear(*_linear_inputs(case, seed))
    if case["kind"] == "append":
        return _exact_append(case, _append_inputs(case, seed))
    return _exact_attention(case, _attention_inputs(case, seed))


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(8)]:
        w = work(c)
        print(c, "%.3g MB, %.3g GFLOP" % (w["bytes"] / 1e6, w["flops"] / 1e9))
