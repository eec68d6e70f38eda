"""Products in 8-bit floating point, and a feed-forward layer of experts on them,
as measured cases.

* ``linear``: a projection in e4m3, activations scaled for each token and block of
  128 channels, weights for each block of 128 x 128: where one scale per
  row is too coarse for the outliers of a row;
* ``route``: the router's logits to the experts of each token and their weights:
  softmax or sigmoid scores, a bias for balance that only takes part in the choice, groups of
  experts of which the best stay, the k best of those, weights made to sum to one;
* ``experts``: a feed-forward layer whose tokens each go through k of E
  gated layers, all in e4m3: rows gathered by expert, gate and up projection, silu(gate) * up,
  down projection, and each token's weighted sum.

Scores decide in 64 bits, equal ones for the lowest expert; an expert of -1
is one that another device holds, and adds nothing.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
TINY = 2.0 ** -126                     # the smallest scale of a block of activations
LARGEST = 4096 * 57344 * 8192          # M * N * K of the largest linear case
PRODUCTS = 4096 * 8 * 4096 * 1024      # T * k * H * I of the largest experts case
WEIGHTS = 128 * 4096 * 1024            # E * H * I of the largest experts case
LOGITS = 16384 * 256


def listed():
    return [
        # one token of one user, a small square projection: launches and latency
        {"name": "linear 1x4096x4096", "kind": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a decode step of a ragged batch through a 70B feed-forward layer: the weights' stream
        {"name": "linear 27x57344x8192", "kind": "linear", "M": 27, "N": 57344, "K": 8192, "dtype": "bf16"},
        # a short prompt of odd length, square projection
        {"name": "linear 203x8192x8192", "kind": "linear", "M": 203, "N": 8192, "K": 8192, "dtype": "fp16"},
        # the largest: long-prompt prefill of a 70B feed-forward layer
        {"name": "linear 4096x57344x8192", "kind": "linear", "M": 4096, "N": 57344, "K": 8192, "dtype": "bf16"},
        # one token, softmax over a few experts
        {"name": "route 1x64", "kind": "route", "T": 1, "E": 64, "k": 6, "dtype": "bf16", "sigmoid": False, "bias": False,
         "groups": 1, "keep": 1, "best": 1, "renorm": True, "scale": 1.0},
        # a prompt, softmax, weights made to sum to one
        {"name": "route 4096x128", "kind": "route", "T": 4096, "E": 128, "k": 8, "dtype": "bf16", "sigmoid": False,
         "bias": False, "groups": 1, "keep": 1, "best": 1, "renorm": True, "scale": 1.0},
        # a batch of long prompts, sigmoid scores with a bias, half of the groups
        {"name": "route 16384x256", "kind": "route", "T": 16384, "E": 256, "k": 8, "dtype": "fp32", "sigmoid": True,
         "bias": True, "groups": 8, "keep": 4, "best": 2, "renorm": True, "scale": 2.5},
        # one token of one user: six experts' weights and no more
        {"name": "experts 1 of 64x2048x1408", "kind": "experts", "T": 1, "E": 64, "k": 6, "H": 2048, "I": 1408,
         "dtype": "bf16", "away": False},
        # a decode step of a ragged batch: most experts' weights for a few rows each
        {"name": "experts 51 of 128x4096x1024", "kind": "experts", "T": 51, "E": 128, "k": 8, "H": 4096, "I": 1024,
         "dtype": "bf16", "away": False},
        # a short prompt, half of the experts on another device
        {"name": "experts 777 of 64x2048x1408", "kind": "experts", "T": 777, "E": 64, "k": 6, "H": 2048, "I": 1408,
         "dtype": "fp16", "away": True},
        # the largest: a long prompt
        {"name": "experts 4096 of 128x4096x1024", "kind": "experts", "T": 4096, "E": 128, "k": 8, "H": 4096, "I": 1024,
         "dtype": "bf16", "away": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of those ranges: every number of rows up to the largest,
    odd widths, several numbers of experts, groups and choices."""
    kind = rng.choice(["linear"] * 4 + ["route"] * 3 + ["experts"] * 4)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "linear":
        step = 16 if rng.random() < 0.15 else 128
        K = max(step, _log(rng, 1024, 16384) // step * step)
        N = _log(rng, 512, 57344)
        if rng.random() < 0.7:
            N = (N + 63) // 64 * 64
        N = min(N, 57344 * 8192 // K)
        return {"kind": kind, "M": min(_log(rng, 1, 4096), LARGEST // (N * K)), "N": N, "K": K, "dtype": dtype}
    if kind == "route":
        E, groups, keep = rng.choice([(8, 1, 1), (60, 1, 1), (64, 1, 1), (64, 8, 3), (128, 1, 1), (160, 8, 3), (256, 1, 1),
                                      (256, 8, 4), (512, 16, 5)])
        sigmoid = rng.random() < 0.5
        return {"kind": kind, "T": _log(rng, 1, min(16384, LOGITS // E)), "E": E, "k": rng.randint(1, 2 if E == 8 else 10),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "sigmoid": sigmoid, "bias": sigmoid and rng.random() < 0.7,
                "groups": groups, "keep": keep, "best": 2 if sigmoid and groups > 1 else 1, "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 1.0, 2.5])}
    E, H, I = rng.choice([(8, 4096, 1792), (16, 2720, 1920), (32, 1024, 512), (60, 2048, 1408), (64, 2048, 1408), (128, 2048, 768),
                          (128, 4096, 1024), (256, 2048, 512)])
    assert E * H * I <= WEIGHTS
    k = rng.randint(1, 2 if E == 8 else 8)
    return {"kind": kind, "T": min(_log(rng, 1, 4096), PRODUCTS // (k * H * I)), "E": E, "k": k, "H": H, "I": I,
            "dtype": dtype, "away": rng.random() < 0.25}


# ------------------------------------------------------------------- inputs
def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _weights(g, *shape):
    """Codes (..., N, K) of normal weights of about 0.02, some rows larger, and
    their scales (..., N / 128, K / 128)."""
    lead, (N, K) = shape[:-2], shape[-2:]
    nb, kb = -(-N // 128), -(-K // 128)
    codes = torch.empty(math.prod(lead), N, K, dtype=E4M3, device=DEV)
    scales = torch.empty(math.prod(lead), nb, kb, device=DEV)
    for e in range(codes.shape[0]):
        for r in range(0, N, 8192):
            n = min(8192, N - r)
            w = torch.randn(-(-n // 128) * 128, kb * 128, generator=g, device=DEV) * 0.02
            w *= torch.exp(0.3 * torch.randn(w.shape[0], 1, generator=g, device=DEV))
            w[n:], w[:, K:] = 0, 0
            w = w.view(-1, 128, kb, 128)
            s = w.abs().amax((1, 3)) / 448
            codes[e, r:r + n] = (w / s[:, None, :, None]).view(-1, kb * 128)[:n, :K].to(E4M3)
            scales[e, r // 128:r // 128 + s.shape[0]] = s
    return codes.view(*lead, N, K), scales.view(*lead, nb, kb)


def _activations(g, rows, K, dtype):
    x = torch.randn(rows, K, generator=g, device=DEV)
    x[:, torch.randperm(K, generator=g, device=DEV)[: K // 100]] *= 20.0     # outlier channels
    return x.to(DTYPES[dtype])


def _linear_inputs(case, seed):
    g = _generator(seed, 31)
    return (_activations(g, case["M"], case["K"], case["dtype"]), *_weights(g, case["N"], case["K"]))


def _route_inputs(case, seed):
    g = _generator(seed, 37)
    T, E = case["T"], case["E"]
    logits = 1.5 * torch.randn(T, E, generator=g, device=DEV) + 0.7 * torch.randn(E, generator=g, device=DEV)
    bias = 0.1 * torch.randn(E, generator=g, device=DEV) if case["bias"] else None
    return logits.to(DTYPES[case["dtype"]]), bias


def _experts_inputs(case, seed):
    """Experts of different popularity; weights that sum to one."""
    g = _generator(seed, 41)
    T, E, k, H, I = (case[n] for n in ("T", "E", "k", "H", "I"))
    every = 2 * E if case["away"] else E
    liked = torch.randn(T, every, generator=g, device=DEV) + 0.7 * torch.randn(every, generator=g, device=DEV)
    top, ids = liked.topk(k, -1)
    ids = torch.where(ids < E, ids, -1).to(torch.int32)
    return (_activations(g, T, H, case["dtype"]), top.softmax(-1), ids, *_weights(g, E, 2 * I, H), *_weights(g, E, H, I))


def prepare(case, seed):
    inputs = {"linear": _linear_inputs, "route": _route_inputs, "experts": _experts_inputs}[case["kind"]]
    return {"case": case, "args": inputs(case, seed)}


# -------------------------------------------------- the operators in plain form
def _plain_quant(x):
    """(..., K) fp32 -> what its codes stand for: a scale for each 128 channels."""
    K = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -K % 128)).unflatten(-1, (-1, 128))
    amax = b.abs().amax(-1, keepdim=True).clamp_min(448 * TINY)
    s = amax / torch.full_like(amax, 448.0)
    # 448 b / amax with one rounding, which leaves halves between codes what they are
    return ((b * 0.875 / amax * 512).to(E4M3).float() * s).flatten(-2)[..., :K]


def _plain_values(codes, scales):
    N, K = codes.shape[-2:]
    s = scales.repeat_interleave(128, -1)[..., :K].repeat_interleave(128, -2)[..., :N, :]
    return codes.float() * s


def _plain_linear(x, wq, ws):
    return (_plain_quant(x.float()) @ _plain_values(wq, ws).t()).to(x.dtype)


def _plain_route(case, logits, bias):
    E, k, G = case["E"], case["k"], case["groups"]
    x = logits.double()
    if case["sigmoid"]:
        score = 1 / (1 + torch.exp(-x))
    else:
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    choice = score if bias is None else score + bias.double()
    if G > 1:
        best = choice.unflatten(-1, (G, E // G)).sort(-1, descending=True)[0][..., :case["best"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True)[1][:, :case["keep"]]
        inside = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = choice.masked_fill(~inside.repeat_interleave(E // G, -1), float("-inf"))
    ids = choice.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    w = score.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"weights": (w * case["scale"]).float(), "ids": ids.to(torch.int32)}


def _plain_experts(x, weights, ids, wq_up, ws_up, wq_down, ws_down):
    T, k = ids.shape
    expert = ids.flatten().long()
    used, slot = expert[expert >= 0].unique(return_inverse=True)
    pair = (expert >= 0).nonzero()[:, 0]
    order = slot.argsort(stable=True)
    pair, slot = pair[order], slot[order]
    count = torch.bincount(slot, minlength=used.numel())
    if pair.numel() == 0:
        return torch.zeros_like(x)
    row = torch.arange(pair.numel(), device=DEV) - (count.cumsum(0) - count)[slot]
    rows = x.new_zeros(used.numel(), int(count.max()), x.shape[1], dtype=torch.float32)
    rows[slot, row] = _plain_quant(x.float())[pair // k]
    gate, up = (rows @ _plain_values(wq_up[used], ws_up[used]).transpose(1, 2)).chunk(2, -1)
    h = _plain_quant(gate / (1 + torch.exp(-gate)) * up)
    out = h @ _plain_values(wq_down[used], ws_down[used]).transpose(1, 2)
    every = x.new_zeros(T * k, x.shape[1], dtype=torch.float32)
    every[pair] = out[slot, row] * weights.flatten()[pair, None]
    return every.view(T, k, -1).sum(1).to(x.dtype)


def run(state):
    case, args = state["case"], state["args"]
    if not own:
        if case["kind"] == "linear":
            return _plain_linear(*args)
        return _plain_route(case, *args) if case["kind"] == "route" else _plain_experts(*args)
    from my_int4 import _C
    if case["kind"] == "linear":
        return _C.fp8_linear(*args)
    if case["kind"] == "route":
        weights, ids = _C.moe_route(args[0], case["k"], bias=args[1], sigmoid=case["sigmoid"], groups=case["groups"],
                                    keep_groups=case["keep"], group_best=case["best"], renorm=case["renorm"],
                                    scale=case["scale"])
        return {"weights": weights, "ids": ids}
    return _C.fp8_experts(*args)


def work(case):
    """Bytes: inputs read once (of the experts those that T * k choices meet), outputs
    written once; operations: the products, of a router one per score and step."""
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * M * K + N * K + N * K // 4096 + 2 * M * N, "flops": 2 * M * N * K}
    T, E, k = case["T"], case["E"], case["k"]
    if case["kind"] == "route":
        return {"bytes": T * E * (4 if case["dtype"] == "fp32" else 2) + 8 * T * k, "flops": T * E * 4}
    H, I, every = case["H"], case["I"], 2 * E if case["away"] else E
    met = E * (1 - (1 - k / every) ** T)
    return {"bytes": int(met * 3 * H * I * (1 + 1 / 4096)) + 4 * T * H + 8 * T * k, "flops": 6 * T * k * H * I * E // every}


# ------------------------------------------------------------ in 64 bits
def _e4m3(x):
    """The nearest value of four exponent and three fraction bits, halves to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_blocks(x):
    """Codes (rows, blocks, 128) and scales (rows, blocks) of x in 64 bits."""
    pad = -x.shape[1] % 128
    b = torch.cat((x.double(), x.new_zeros(x.shape[0], pad, dtype=torch.float64)), 1).view(x.shape[0], -1, 128)
    amax = b.abs().amax(2).clamp_min(448 * TINY)
    return _e4m3(b * 448 / amax[..., None]), amax / 448


def _exact_product(x, wq, ws):
    """Block by block of 128 channels, weights' scales applied to the partial sums."""
    q, s = _exact_blocks(x)
    N, K = wq.shape
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=DEV)
    for b in range(s.shape[1]):
        w = wq[:, 128 * b:128 * b + 128].float().double()
        part = q[:, b, :w.shape[1]].contiguous() @ w.t().contiguous()
        y += part * s[:, b, None] * ws[:, b].double().repeat_interleave(128)[:N]
    return y


def _exact_route(case, logits, bias):
    x = logits.double()
    score = torch.sigmoid(x) if case["sigmoid"] else torch.softmax(x, -1)
    choice = score.clone() if bias is None else score + bias.double()
    E, G = case["E"], case["groups"]
    if G > 1:
        of = choice.view(-1, G, E // G).topk(case["best"], 2).values.sum(2)
        better = (of[:, None] > of[:, :, None]) | ((of[:, None] == of[:, :, None]) & torch.ones(G, G, device=DEV).tril(-1).bool())
        out = better.sum(2) >= case["keep"]
        choice[out.repeat_interleave(E // G, 1)] = -math.inf
    ids = []
    for _ in range(case["k"]):
        at = (choice == choice.amax(1, keepdim=True)).int().argmax(1)          # the first of the largest
        ids.append(at)
        choice[torch.arange(at.numel(), device=DEV), at] = -math.inf
    ids = torch.stack(ids, 1)
    w = score.gather(1, ids)
    return {"weights": (w / w.sum(1, keepdim=True) if case["renorm"] else w) * case["scale"], "ids": ids.to(torch.int32)}


def _exact_experts(x, weights, ids, wq_up, ws_up, wq_down, ws_down):
    """Expert by expert."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    I = wq_down.shape[2]
    for e in range(wq_up.shape[0]):
        token, choice = (ids == e).nonzero(as_tuple=True)
        if token.numel():
            a = _exact_product(x[token], wq_up[e], ws_up[e])
            h = a[:, :I] * torch.sigmoid(a[:, :I]) * a[:, I:]
            y.index_add_(0, token, _exact_product(h, wq_down[e], ws_down[e]) * weights[token, choice].double()[:, None])
    return y


def exact(case, seed):
    if case["kind"] == "linear":
        return _exact_product(*_linear_inputs(case, seed))
    if case["kind"] == "route":
        return _exact_route(case, *_route_inputs(case, seed))
    return _exact_experts(*_experts_inputs(case, seed))


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(s)) for s in range(8)]:
        w = work(c)
        print(c, "%.3g MB, %.3g GFLOP" % (w["bytes"] / 1e6, w["flops"] / 1e9))
