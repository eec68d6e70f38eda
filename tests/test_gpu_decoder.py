"""The decoder layer that runs the 8-bit operators and the W4A4 step together."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def layer_of(seed, K, Hq, Hkv, D, F, dev):
    from my_int4 import _C
    from my_int4.decoder import DecoderLayer, quant_weight_int8
    g = torch.Generator().manual_seed(seed)
    w = {n: torch.randn(*s, generator=g) / s[1] ** 0.5 for n, s in
         {"qkv": ((Hq + 2 * Hkv) * D, K), "out": (K, Hq * D), "up": (F, K), "down": (K, F)}.items()}
    t = torch.eye(32).repeat(K // 32, 1, 1).bfloat16()
    up = (t.to(dev), *_C.quant_int4(w["up"].bfloat16().to(dev)))
    q8 = {n: tuple(t.to(dev) for t in quant_weight_int8(w[n])) for n in ("qkv", "out", "down")}
    norm = 1 + 0.1 * torch.randn(2, K, generator=g)
    return DecoderLayer(Hq, Hkv, q8["qkv"], q8["out"], up, q8["down"], norm[0].to(dev), norm[1].to(dev)), w, norm


def plain_attention_half(x, w, norm, Hq, Hkv, D, cos_sin, upto):
    """The attention half of one sequence in fp64 and with nothing quantized; rows `upto` on."""
    x = x.double()
    h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * norm.double()
    q, k, v = (h @ w["qkv"].double().t()).view(x.shape[0], -1, D).split([Hq, Hkv, Hkv], 1)
    c, s = cos_sin.double()[:x.shape[0], None].chunk(2, -1)

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * D ** -0.5
    s = s.masked_fill(torch.ones(x.shape[0], x.shape[0]).triu(1).bool(), float("-inf"))
    o = torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(x.shape[0], -1)
    return (o @ w["out"].double().t())[upto:]


def test_layer_prefill_then_decode(dev):
    """Prompts of different lengths, then tokens one by one in a replayed graph.
    The attention half against the same in fp64 without any quantization: 8-bit
    activations, keys, values and weights are each off by about 1% rms (a uniform
    error of a 127th of the largest of some thousand normal values, 3 to 4 of their
    sigma: 0.9%); five such steps in quadrature are 2%, the gate is twice that."""
    from my_int4.chain import graphed
    from my_int4.decoder import KV8Cache, rotation_table
    K, Hq, Hkv, D, F, steps = 512, 8, 2, 64, 1024, 5
    layer, w, norm = layer_of(1, K, Hq, Hkv, D, F, dev)
    cs = rotation_table(256, D, device=dev)
    lens0 = [37, 1, 130]
    g = torch.Generator().manual_seed(2)
    xs = [torch.randn(m + steps, K, generator=g).bfloat16() for m in lens0]
    cache = KV8Cache(16, Hkv, D, page_size=32, device=dev)
    host = torch.full((3, 6), -1, dtype=torch.int32)
    for b, m in enumerate(lens0):
        cache.grow(host, b, m + steps)
    table = host.to(dev)
    lens = torch.tensor(lens0, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 37, 38, 168], dtype=torch.int32, device=dev)
    x = torch.cat([t[:m] for t, m in zip(xs, lens0)]).to(dev)
    half = layer.attention(x, cache, cs, table, lens, cu).cpu().double() - x.cpu().double()
    at = 0
    for t, m in zip(xs, lens0):
        ref = plain_attention_half(t[:m], w, norm[0], Hq, Hkv, D, cs.cpu(), 0)
        assert float((half[at:at + m] - ref).norm() / ref.norm()) < 0.04
        at += m
    full = layer.step(x, cache, cs, table, lens, cu)                # again: the cache does not change
    assert full.shape == x.shape and bool(torch.isfinite(full.float()).all())

    x1 = torch.stack([t[m] for t, m in zip(xs, lens0)]).to(dev)
    lens += 1
    state = [t.clone() for t in cache.tensors()]
    graph, y = graphed(lambda: (layer.attention(x1, cache, cs, table, lens), layer.step(x1, cache, cs, table, lens)))
    for t, s in zip(cache.tensors(), state):
        t.copy_(s)
    lens -= 1
    for i in range(steps):
        x1.copy_(torch.stack([t[m + i] for t, m in zip(xs, lens0)]))
        lens += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[1], layer.step(x1, cache, cs, table, lens))
        for b, (t, m) in enumerate(zip(xs, lens0)):
            ref = plain_attention_half(t[:m + i + 1], w, norm[0], Hq, Hkv, D, cs.cpu(), m + i)
            got = y[0][b].cpu().double() - x1[b].cpu().double()
            assert float((got - ref[0]).norm() / ref.norm()) < 0.04, (i, b)


def test_cache_pages(dev):
    from my_int4.decoder import KV8Cache
    c = KV8Cache(4, 1, 64, page_size=16, device=dev)
    t = torch.full((2, 3), -1, dtype=torch.int32)
    assert c.grow(t, 0, 17) == 2 and c.grow(t, 0, 20, 2) == 2 and c.grow(t, 1, 1) == 1 and len(c.free) == 1
    with pytest.raises(MemoryError):
        c.grow(t, 1, 48, 1)
    with pytest.raises(ValueError):
        c.grow(t, 1, 49, 1)
    assert len(set(t[t >= 0].tolist())) == 3
    c.release(t, 0, 2)
    assert len(c.free) == 3 and int(t[0].max()) == -1
