"""The router and the experts' layers on the GPU: choices equal, weights and
outputs within the bounds of their roundings."""
from __future__ import annotations

import math

import pytest
import torch

import _fp8 as plain

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check_route(_C, x, k, bias=None, sigmoid=False, groups=1, keep=1, best=1, renorm=True, scale=1.0):
    w, ids = _C.moe_route(x, k, bias=bias, sigmoid=sigmoid, groups=groups, keep_groups=keep, group_best=best, renorm=renorm,
                          scale=scale)
    ew, eids = plain.route(x.reshape(-1, x.shape[-1]), k, bias, sigmoid, groups, keep, best, renorm, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.shape == ids.shape == (*x.shape[:-1], k)
    assert torch.equal(ids.cpu().long().reshape(eids.shape), eids)
    got = w.cpu().double().reshape(ew.shape)
    nan = torch.isnan(ew)
    assert torch.equal(torch.isnan(got), nan)
    # one rounding to fp32 (denormals kept), 64-bit steps before
    assert bool(((got - ew).abs() <= 1.01 * 2.0 ** -24 * ew.abs() + 2.0 ** -150)[~nan].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,k,groups,keep,best", [
    (1, 1, 1, 1, 1, 1), (3, 2, 2, 1, 1, 1), (5, 7, 3, 1, 1, 1), (9, 8, 2, 1, 1, 1), (33, 60, 4, 1, 1, 1), (64, 64, 6, 1, 1, 1),
    (17, 64, 64, 1, 1, 1), (40, 128, 8, 1, 1, 1), (12, 160, 6, 8, 3, 1), (50, 256, 8, 8, 4, 2), (7, 256, 10, 64, 9, 2),
    (6, 300, 5, 60, 5, 2), (5, 1000, 12, 40, 3, 1), (4, 1024, 17, 1, 1, 1), (4, 512, 9, 16, 5, 2), (3, 513, 3, 3, 2, 1)])
def test_route(dev, dtype, T, E, k, groups, keep, best):
    from my_int4 import _C
    g = gen(T + E + k)
    x = (1.5 * torch.randn(T, E, generator=g)).to(dtype).to(dev)
    bias = (0.1 * torch.randn(E, generator=g)).to(dev)
    check_route(_C, x, k, None, False, groups, keep, best, True, 1.0)
    check_route(_C, x, k, bias, True, groups, keep, best, True, 2.5)
    check_route(_C, x, k, bias, False, groups, keep, best, False, 1.0)
    check_route(_C, x, k, None, True, groups, keep, best, False, -0.5)


@pytest.mark.parametrize("E,groups,keep", [(64, 1, 1), (128, 8, 3), (1000, 40, 9)])
def test_route_ties(dev, E, groups, keep):
    # few different values: ties within lanes, across lanes and between groups
    from my_int4 import _C
    g = gen(E)
    x = torch.randint(-2, 3, (40, E), generator=g).to(dev).bfloat16()
    bias = torch.randint(0, 2, (E,), generator=g).float().to(dev)
    for b in (None, bias):
        for sigmoid in (False, True):
            for best in (1, 2):
                check_route(_C, x, 8, b, sigmoid, groups, keep, best)
    x[0] = 0.0
    x[1] = -0.0
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    check_route(_C, x, 8, None, True, groups, keep, 1)


def test_route_values_at_a_border(dev):
    # scores that differ in the 40th bit only, and equal ones
    from my_int4 import _C
    x = torch.full((4, 64), 3.0)
    x[0, 40] = 3.0 + 2.0 ** -22
    x[1] = 20.0 + torch.arange(64) * 2.0 ** -19
    x[2] = torch.arange(64).flip(0) * 2.0 ** -30
    bias = torch.zeros(64)
    bias[50] = 2.0 ** -40
    for b in (None, bias.to(dev)):
        check_route(_C, x.to(dev), 5, b, True)
    check_route(_C, x[:2].to(dev), 5, None, False)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (8, 2, 1), (8, 2, 2)])
def test_route_masked_rows(dev, sigmoid, groups, keep, best):
    from my_int4 import _C
    g = gen(3)
    x = torch.randn(10, 64, generator=g)
    x[0] = -math.inf
    x[1, 3:] = -math.inf                                        # fewer than k left
    x[2] = torch.finfo(torch.float32).min
    x[3, 5] = math.inf
    x[4, 9] = math.nan
    x[5] = math.nan
    x[6] = math.inf
    x[7, ::2] = torch.finfo(torch.float32).min
    x[8] = 1e30
    x[8, 11] = -1e30
    for renorm in (False, True):
        check_route(_C, x.to(dev), 8, None, sigmoid, groups, keep, best, renorm)
        check_route(_C, x.to(dev), 8, torch.linspace(-1, 1, 64, device=dev), sigmoid, groups, keep, best, renorm)


def test_route_layouts(dev):
    from my_int4 import _C
    x = torch.randn(30, 64, generator=gen(4)).to(dev)
    w, ids = _C.moe_route(x, 6)
    wide = torch.full((30, 71), math.nan, device=dev)
    for at in (0, 1, 7):
        wide[:, at:at + 64] = x
        a, b = _C.moe_route(wide[:, at:at + 64], 6)
        assert torch.equal(a, w) and torch.equal(b, ids)
    for y, shape in ((x.t().contiguous().t(), (30, 6)), (x.view(5, 6, 64), (5, 6, 6))):
        a, b = _C.moe_route(y, 6)
        assert a.shape == shape and torch.equal(a.view(30, 6), w) and torch.equal(b.view(30, 6), ids)
    a, b = _C.moe_route(x[0], 6)
    assert a.shape == (6,) and torch.equal(a, w[0]) and torch.equal(b, ids[0])
    a, b = _C.moe_route(x[:1].expand(9, 64), 6)
    assert torch.equal(a, w[:1].expand(9, 6)) and torch.equal(b, ids[:1].expand(9, 6))
    assert _C.moe_route(x[:0], 6)[0].shape == (0, 6)


def test_route_more_rows_than_a_launch(dev):
    # 2^26 + 5 rows: three launches of 2^25 rows at most, the last of a few
    from my_int4 import _C
    T = (1 << 26) + 5
    x = torch.zeros(T, 2, dtype=torch.bfloat16, device=dev)
    x[:, 1] = torch.arange(T, device=dev) % 7 - 3
    w, ids = _C.moe_route(x, 1, sigmoid=True, renorm=False)
    assert torch.equal(ids[:, 0], (x[:, 1] > 0).int())
    few = torch.cat((torch.arange(9), torch.arange((1 << 25) - 3, (1 << 25) + 3), torch.arange(T - 9, T))).to(dev)
    check_route(_C, x[few], 1, None, True, 1, 1, 1, False)
    assert torch.equal(w[few], _C.moe_route(x[few], 1, sigmoid=True, renorm=False)[0])


def case(seed, T, E, k, H, I, dev, dtype=torch.bfloat16, away=0.0):
    g = gen(seed)
    x = torch.randn(T, H, generator=g).to(dtype)
    score = torch.randn(T, E, generator=g) + torch.randn(E, generator=g)
    top, ids = score.topk(k, -1)
    ids = torch.where(torch.rand(T, k, generator=g) < away, -1, ids).to(torch.int32)
    up, down = plain.weights(g, E, 2 * I, H), plain.weights(g, E, H, I)
    # outputs of about one
    return [t.to(dev) for t in (x, top.softmax(-1), ids, up[0], up[1] * (16 / H ** 0.5), down[0], down[1] * (2.0 ** -4 / I ** 0.5))]


def check_experts(_C, args):
    y = _C.fp8_experts(*args)
    assert y.shape == args[0].shape and y.dtype == args[0].dtype
    within(y, args)
    return y


def within(y, args):
    """The bound of one of the three ways: all products exact (few tokens); the down projection's cut; both's, and an
    expert's rows kept in fp16.  Each says something: it is a small part of the outputs (a single token whose one
    open code lets all of a row's cut products count: 7 * 2^-13 * sum |h w| / |y|, some 2% for hundreds of terms, and the code)."""
    ratios = []
    for way in ((False, False), (False, True), (True, True, 2.0 ** -11)):
        ref, err = plain.experts(*args, *way)
        assert float(err.norm()) <= 0.1 * float(ref.norm())
        ratios.append(plain.off(y, ref, err, y.dtype))
    assert min(ratios) <= 1, ratios


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 1, 1, 16, 128), (1, 8, 2, 256, 128), (1, 64, 6, 1024, 384), (2, 16, 4, 272, 128), (4, 8, 8, 512, 256),
                                       (5, 40, 3, 1040, 256), (33, 16, 2, 512, 384), (64, 64, 8, 768, 128), (200, 8, 2, 640, 256),
                                       (300, 4, 1, 400, 128), (777, 16, 4, 256, 256), (513, 3, 2, 1024, 512), (1500, 2, 1, 512, 128),
                                       (2000, 6, 3, 656, 640), (3100, 40, 2, 128, 2048)])
def test_experts(dev, dtype, T, E, k, H, I):
    from my_int4 import _C
    args = case(T + E + H, T, E, k, H, I, dev, dtype)
    y = check_experts(_C, args)
    assert torch.equal(y, _C.fp8_experts(*args))


@pytest.mark.parametrize("T", [1, 3, 50, 400])
def test_experts_elsewhere(dev, T):
    # ids that name no expert here, whole tokens and whole experts without any
    from my_int4 import _C
    args = case(T, T, 12, 3, 384, 128, dev, away=0.6)
    args[2][0] = torch.tensor([-1, 12, 2 ** 31 - 1], dtype=torch.int32)
    args[2][args[2] == 4] = -(2 ** 31)
    y = check_experts(_C, args)
    assert not bool(y[0].any())
    args[2].fill_(-1)
    assert not bool(_C.fp8_experts(*args).any())


def test_experts_one_takes_all(dev):
    from my_int4 import _C
    for T in (2, 70, 600):
        args = case(T, T, 32, 2, 256, 128, dev)
        args[2].fill_(31)                                       # the same expert twice
        check_experts(_C, args)


def test_experts_more_than_one_run(dev):
    # 70000 pairs: more than are taken at once; each token as if it were alone with others
    from my_int4 import _C
    args = case(1, 17500, 4, 4, 128, 128, dev)
    y = _C.fp8_experts(*args)
    for a, b in ((0, 300), (16300, 16500), (17400, 17500)):
        part = [args[0][a:b], args[1][a:b].contiguous(), args[2][a:b].contiguous(), *args[3:]]
        within(y[a:b], part)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_experts_layouts(dev, T):
    from my_int4 import _C
    args = case(T, T, 8, 2, 272, 128, dev)
    x = args[0]
    y = _C.fp8_experts(*args)
    wide = torch.full((T, 272 + 40), math.nan, dtype=x.dtype, device=dev)
    for at in (0, 8, 3):
        wide[:, at:at + 272] = x
        assert torch.equal(_C.fp8_experts(wide[:, at:at + 272], *args[1:]), y)
    assert torch.equal(_C.fp8_experts(x.view(T, 1, 272), args[1].view(T, 1, 2), args[2].view(T, 1, 2), *args[3:]), y.view(T, 1, 272))
    none = _C.fp8_experts(x[:0], args[1][:0], args[2][:0], *args[3:])
    assert none.shape == (0, 272)


def test_experts_non_finite_tokens_stay_alone(dev):
    from my_int4 import _C
    for T in (3, 200):
        args = case(9, T, 6, 2, 256, 128, dev)
        clean = _C.fp8_experts(*args)
        args[0][1, 200] = math.inf
        y = _C.fp8_experts(*args)
        assert torch.isnan(y[1]).all()
        keep = [t for t in range(T) if t != 1]
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E", [(1300, 64), (2700, 8)])
def test_experts_non_finite_tokens_stay_alone_from_tile_to_tile(dev, T, E, dtype):
    # more tiles than workgroups, one after another
    from my_int4 import _C
    args = case(10, T, E, 2, 2048, 1024, dev, dtype=dtype)
    clean = _C.fp8_experts(*args)
    args[0][::9, 200] = math.inf
    y = _C.fp8_experts(*args)
    bad = torch.arange(T, device=dev) % 9 == 0
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], clean[~bad])


def test_route_and_experts_in_a_graph(dev):
    from my_int4 import _C
    for T in (1, 24, 300):
        args = case(T, T, 16, 4, 512, 256, dev)
        logits = torch.randn(T, 16, generator=gen(7)).to(dev)

        def layer():
            w, ids = _C.moe_route(logits, 4, sigmoid=True, groups=4, keep_groups=2, group_best=2)
            return w, ids, _C.fp8_experts(args[0], w, ids, *args[3:])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        for i in range(3):
            if i:
                logits.copy_(torch.randn(T, 16, generator=gen(70 + i)).to(dev))
                args[0].copy_(torch.randn(T, 512, generator=gen(80 + i)).to(dev))
            expect = layer()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, expect))
            within(out[2], [args[0], *out[:2], *args[3:]])


def test_refusals(dev):
    from my_int4 import _C
    x = torch.zeros(4, 64, device=dev)
    bad = [
        ("bf16, fp16 or fp32", lambda: _C.moe_route(x.double(), 2)),
        ("CUDA", lambda: _C.moe_route(x.cpu(), 2)),
        ("1 to 1024 experts", lambda: _C.moe_route(torch.zeros(1, 1025, device=dev), 2)),
        ("divide", lambda: _C.moe_route(x, 2, groups=5)),
        ("keep_groups", lambda: _C.moe_route(x, 2, groups=4, keep_groups=5)),
        ("group_best", lambda: _C.moe_route(x, 2, groups=4, keep_groups=2, group_best=3)),
        ("group_best", lambda: _C.moe_route(x, 2, groups=64, keep_groups=2, group_best=2)),
        ("k must be", lambda: _C.moe_route(x, 0)),
        ("k must be", lambda: _C.moe_route(x, 33, groups=4, keep_groups=2)),
        ("k must be", lambda: _C.moe_route(torch.zeros(1, 100, device=dev), 65)),
        ("scale", lambda: _C.moe_route(x, 2, scale=math.inf)),
        ("one value per expert", lambda: _C.moe_route(x, 2, bias=torch.zeros(63, device=dev))),
        ("fp32", lambda: _C.moe_route(x, 2, bias=torch.zeros(64, device=dev, dtype=torch.half))),
    ]
    a = case(0, 3, 4, 2, 256, 128, dev)

    def change(i, t):
        return [*a[:i], t, *a[i + 1:]]

    bad += [(text, lambda b=b: _C.fp8_experts(*b)) for text, b in [
        ("bf16 or fp16", change(0, a[0].float())),
        ("columns", change(0, a[0][:, :128].contiguous())),
        ("tokens, k", change(1, a[1][:2].contiguous())),
        ("fp32", change(1, a[1].half())),
        ("int32", change(2, a[2].long())),
        ("float8_e4m3fn", change(3, a[3].float())),
        ("3D", change(3, a[3][0])),
        ("one scale per 128", change(4, a[4][:, :1].contiguous())),
        ("w_up must be", change(3, a[3][:, :128].contiguous())[:4] + [a[4][:, :1].contiguous(), *a[5:]]),
        ("one scale per 128", change(6, a[6][:3].contiguous())),
        ("CUDA", change(2, a[2].cpu())),
    ]]
    for text, call in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
