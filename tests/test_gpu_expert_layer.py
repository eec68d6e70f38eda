"""A decoder layer whose feed-forward half is a layer of experts."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def experts_of(g, E, k, K, I, dev, shared=True, **kw):
    from my_int4.decoder import ExpertLayer, quant_weight_fp8
    w = {"router": torch.randn(E, K, generator=g) / K ** 0.5, "up": torch.randn(E, 2 * I, K, generator=g) / K ** 0.5,
         "down": torch.randn(E, K, I, generator=g) / I ** 0.5, "up1": torch.randn(2 * I, K, generator=g) / K ** 0.5,
         "down1": torch.randn(K, I, generator=g) / I ** 0.5, "bias": 0.1 * torch.randn(E, generator=g)}

    def q(t):
        return tuple(a.to(dev) for a in quant_weight_fp8(t))

    layer = ExpertLayer(w["router"].to(dev), k, q(w["up"]), q(w["down"]), bias=w["bias"].to(dev), sigmoid=True, groups=4, keep_groups=2,
                        group_best=2, scale=1.5, shared=(q(w["up1"]), q(w["down1"])) if shared else None, **kw)
    return layer, w


def gated(x, up, down):
    gate, value = (x @ up.double().t()).chunk(2, -1)
    return (torch.nn.functional.silu(gate) * value) @ down.double().t()


def plain_experts(x, w, layer, shared=True, only=None):
    """In fp64, nothing quantized, but for the choice, which is that of the same fp32 logits."""
    import _fp8 as plain
    logits = torch.nn.functional.linear(x.float(), layer.router)
    wt, ids = plain.route(logits, layer.k, layer.bias, True, 4, 2, 2, True, 1.5)
    x = x.double().cpu()
    y = gated(x, w["up1"], w["down1"]) if shared else torch.zeros_like(x)
    for e in range(w["up"].shape[0]) if only is None else only:
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            y[t] += wt[t, j][:, None] * gated(x[t], w["up"][e], w["down"][e])
    return y


# Rounding to e4m3 is off by up to 2^-4 of a value, evenly spread within steps that are 2^-4 to 2^-3 of it: 2 to 3.6% of
# the root mean square.  Inputs and weights of a product each contribute that much: 3.6% sqrt(2) for each of gate and up,
# together 7.2%, with the hidden values' and the last weights' 3.6% each 8.8%.  The gate is 1.25 times that.
GATE = 0.11


@pytest.mark.parametrize("T", [1, 3, 60, 500])
def test_expert_layer(dev, T):
    g = torch.Generator().manual_seed(T)
    layer, w = experts_of(g, 16, 4, 256, 384, dev)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(T, 256, generator=g).to(dtype).to(dev)
        y = layer(x)
        ref = plain_experts(x, w, layer)
        assert y.shape == x.shape and y.dtype == dtype
        assert float((y.double().cpu() - ref).norm() / ref.norm()) < GATE


def test_parts_of_the_experts_add_up(dev):
    from my_int4.decoder import ExpertLayer
    g = torch.Generator().manual_seed(5)
    layer, w = experts_of(g, 16, 4, 256, 128, dev, shared=False)
    x = torch.randn(70, 256, generator=g).bfloat16().to(dev)
    total = torch.zeros(70, 256, dtype=torch.float64, device=dev)
    for at in (0, 4, 10):
        n = {0: 4, 4: 6, 10: 6}[at]
        part = ExpertLayer(**{**layer.__dict__, "first": at, "up": tuple(t[at:at + n].contiguous() for t in layer.up),
                              "down": tuple(t[at:at + n].contiguous() for t in layer.down)})
        y = part(x)
        ref = plain_experts(x, w, layer, False, range(at, at + n))
        assert float((y.double().cpu() - ref).norm() / ref.norm()) < GATE
        total += y.double()
    whole = layer(x).double()
    # each part and the whole are rounded to bf16: 2^-8 of each value
    assert float((total - whole).norm() / whole.norm()) < 2 * 2.0 ** -8


def test_decoder_layer_with_experts(dev):
    """Prompts, then tokens one by one in a replayed graph, against eager calls; the feed-forward half against the
    experts on the attention half's output."""
    from my_int4.chain import graphed
    from my_int4.decoder import DecoderLayer, KV8Cache, _norm, quant_weight_int8, rotation_table
    K, Hq, Hkv, D, steps = 256, 4, 2, 64, 4
    g = torch.Generator().manual_seed(7)
    experts, w = experts_of(g, 16, 4, K, 256, dev)
    q8 = [tuple(t.to(dev) for t in quant_weight_int8(torch.randn(*s, generator=g) / s[1] ** 0.5)) for s in (((Hq + 2 * Hkv) * D, K), (K, Hq * D))]
    norm = 1 + 0.1 * torch.randn(2, K, generator=g)
    layer = DecoderLayer(Hq, Hkv, q8[0], q8[1], None, None, norm[0].to(dev), norm[1].to(dev), experts=experts)
    cs, lens0 = rotation_table(256, D, device=dev), [37, 1, 130]
    xs = [torch.randn(m + steps, K, generator=g).bfloat16() for m in lens0]
    cache = KV8Cache(24, Hkv, D, page_size=16, device=dev)
    host = torch.full((3, 10), -1, dtype=torch.int32)
    for b, m in enumerate(lens0):
        cache.grow(host, b, m + steps)
    table, lens = host.to(dev), torch.tensor(lens0, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 37, 38, 168], dtype=torch.int32, device=dev)
    x = torch.cat([t[:m] for t, m in zip(xs, lens0)]).to(dev)
    half = layer.attention(x, cache, cs, table, lens, cu)
    full = layer.step(x, cache, cs, table, lens, cu)
    ref = plain_experts(_norm(half, layer.norm2), w, experts)
    got = full.double().cpu() - half.double().cpu()
    assert float((got - ref).norm() / ref.norm()) < GATE + 2.0 ** -8 * float(full.double().norm()) / float(ref.norm())
    x1 = torch.stack([t[m] for t, m in zip(xs, lens0)]).to(dev)
    lens += 1
    state = [t.clone() for t in cache.tensors()]
    graph, y = graphed(lambda: layer.step(x1, cache, cs, table, lens))
    for t, s in zip(cache.tensors(), state):
        t.copy_(s)
    lens -= 1
    for i in range(steps):
        x1.copy_(torch.stack([t[m + i] for t, m in zip(xs, lens0)]))
        lens += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer.step(x1, cache, cs, table, lens))
