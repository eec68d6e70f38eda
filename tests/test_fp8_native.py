"""CPU checks of the e4m3 operators' and the router's host side: bad arguments are refused and empty
work succeeds before any device is touched; workspace sizes and plans are host only; the torch module
exposes the operators and refuses CPU tensors; the weights' quantizer; the tests' own oracle."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import _fp8 as plain

INVALID = 1
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def capi():
    from wush_int4_kernel_amd import capi as c
    c.load()
    return c


def test_fp8_arguments(capi):
    lib = capi.load()
    quant, gemm, linear = lib.wush_quant_fp8_block, lib.wush_gemm_fp8, lib.wush_linear_fp8
    assert quant(None, 0, None, None, 0, 64, 64, None) == 0
    for args in [(None, 0, P(16), P(16), 1, 64, 64), (P(16), 2, P(16), P(16), 1, 64, 64), (P(8), 0, P(16), P(16), 1, 64, 64),
                 (P(16), 0, P(8), P(16), 1, 64, 64), (P(16), 0, P(16), P(16), 1, 40, 40), (P(16), 0, P(16), P(16), 1, 131072, 131072),
                 (P(16), 0, P(16), P(16), 2, 64, 60), (P(16), 0, P(16), P(16), 2, 64, -64), (P(16), 0, P(16), P(16), -1, 64, 64),
                 (P(16), 0, P(16), P(2), 1, 64, 64), (P(16), 0, P(16), P(16), 1, 0, 64), (P(16), 0, P(16), P(16), 1 << 27, 64, 64)]:
        assert quant(*args, None) == INVALID, args
    ok = [P(16)] * 5
    assert gemm(*[None] * 5, 0, 0, 8, 64, None, 0, None) == 0 and gemm(*[None] * 5, 0, 8, 0, 64, None, 0, None) == 0
    for M in (1, 5, 300):
        for args in [(*ok, 2, M, 8, 64), (*ok, 0, M, 8, 40), (*ok, 0, M, 8, 131072), (*ok, 0, -M, 8, 64), (None, *ok[1:], 0, M, 8, 64),
                     (P(8), *ok[1:], 0, M, 8, 64), (*ok[:2], P(8), *ok[3:], 0, M, 8, 64), (*ok[:4], P(1), 0, M, 7, 64), (*ok, 0, M, 8, 0),
                     (*ok[:4], P(8), 0, M, 8, 64), (P(16), P(2), *ok[2:], 0, M, 8, 64), (*ok[:3], P(2), P(16), 0, M, 8, 64),
                     (*ok, 0, M, 1 << 27, 64), (*ok, 0, 1 << 27, 8, 64)]:
            assert gemm(*args, None, 0, None) == INVALID, args
    assert linear(None, 64, None, None, None, 0, 0, 8, 64, None, 0, None) == 0
    assert lib.wush_linear_fp8_workspace_bytes(4, 8, 64) == 0
    need = lib.wush_linear_fp8_workspace_bytes(20, 8, 272)
    assert need >= 20 * 272 + 20 * 3 * 4
    for args in [(P(16), 272, P(16), need - 1), (P(16), 272, None, need), (P(16), 272, P(8), need), (P(16), 268, P(16), need), (P(8), 272, P(16), need)]:
        assert linear(args[0], args[1], P(16), P(16), P(16), 0, 20, 8, 272, args[2], args[3], None) == INVALID, args
    assert linear(P(16), 60, P(16), P(16), P(16), 0, 2, 8, 64, None, 0, None) == INVALID
    assert lib.wush_gemm_fp8_workspace_bytes(0, 8, 64) == 0 == lib.wush_linear_fp8_workspace_bytes(0, 8, 64)


def test_plan_queries(capi):
    lib = capi.load()
    plan = (ctypes.c_int32 * 4)()
    for args in [(0, 8, 64), (1, 0, 64), (1, 8, 40), (1, 8, 131072), (1, 8, 0)]:
        assert lib.wush_gemm_fp8_plan(*args, 0, plan) == INVALID, args
    assert lib.wush_gemm_fp8_plan(1, 8, 64, 0, None) == INVALID
    for M, K in ((1, 32768), (2, 16384), (3, 8192), (4, 8192)):
        assert capi.gemm_fp8_plan(M, 4096, K)[0] == capi.FP8_DOT
        assert capi.gemm_fp8_plan(M, 4096, K + 16)[0] == capi.FP8_TILES
    kernel, _, _, slices = capi.gemm_fp8_plan(13, 4096, 8192)
    assert kernel == capi.FP8_TILES and slices > 1 and capi.gemm_fp8_plan(13, 4096, 8192, 0)[3] == 1
    assert lib.wush_gemm_fp8_workspace_bytes(13, 4096, 8192) == slices * 13 * 4096 * 4
    # tiles of 64 and 128 x 256 store 16 bytes at a time
    assert {capi.gemm_fp8_plan(M, 57344, 8192)[1:3] for M in (40, 100)} == {(64, 256), (128, 256)}
    assert all(capi.gemm_fp8_plan(M, 57343, 8192)[2] < 256 or capi.gemm_fp8_plan(M, 57343, 8192)[1] == 256 for M in (40, 100, 500))


def test_route_arguments(capi):
    lib = capi.load()

    def route(logits=P(16), dtype=0, stride=64, bias=None, rows=3, experts=64, weights=P(16), ids=P(16), choice=True, **kw):
        c = capi.MoeChoice(**{**dict(k=4, groups=1, keep_groups=1, group_best=1, sigmoid=0, renorm=1, scale=1.0), **kw})
        return lib.wush_moe_route(logits, dtype, stride, bias, rows, experts, ctypes.byref(c) if choice else None, weights, ids, None)

    assert route(rows=0, logits=None) == 0
    for kw in [dict(choice=False), dict(logits=None), dict(dtype=3), dict(stride=-1), dict(bias=P(2)), dict(rows=-1), dict(experts=0),
               dict(experts=1025), dict(weights=None), dict(ids=None), dict(weights=P(2)), dict(k=0), dict(k=65), dict(k=5, experts=4),
               dict(groups=0), dict(groups=3), dict(groups=65, experts=65), dict(groups=8, keep_groups=9), dict(keep_groups=0),
               dict(groups=8, keep_groups=2, k=17), dict(group_best=0), dict(group_best=3), dict(group_best=2, experts=64, groups=64),
               dict(scale=math.inf), dict(scale=math.nan), dict(logits=P(17)), dict(logits=P(18), dtype=2)]:
        assert route(**kw) == INVALID, kw


def test_experts_arguments(capi):
    lib = capi.load()
    size = lib.wush_moe_experts_fp8_workspace_bytes
    assert size(0, 2, 8, 256, 128, 0) == 0 == size(1, 2, 8, 250, 128, 0) == size(1, 2, 8, 256, 100, 0) == size(1, 2, 2000, 256, 128, 0)

    def run(T=3, k=2, E=8, H=256, I=128, dtype=0, stride=256, ws=P(256), wsb=None, **kw):
        a = dict(x=P(16), weights=P(16), ids=P(16), w_up=P(16), s_up=P(16), w_down=P(16), s_down=P(16), y=P(16), **{})
        a.update(kw)
        need = size(T, k, E, H, I, dtype)
        return lib.wush_moe_experts_fp8(a["x"], dtype, stride, a["weights"], a["ids"], a["w_up"], a["s_up"], a["w_down"], a["s_down"],
                                        a["y"], T, k, E, H, I, ws, need if wsb is None else need + wsb, None)

    assert run(T=0, x=None) == 0
    for T in (3, 400):
        for kw in [dict(x=None), dict(x=P(8)), dict(weights=None), dict(ids=P(2)), dict(w_up=P(8)), dict(s_up=None), dict(w_down=None),
                   dict(s_down=P(1)), dict(y=None), dict(y=P(1)), dict(k=0), dict(k=65), dict(E=0), dict(E=1025), dict(H=250), dict(I=64),
                   dict(I=0), dict(dtype=2), dict(stride=252), dict(stride=-256), dict(ws=None), dict(ws=P(8)), dict(wsb=-1)]:
            assert run(T=T, **kw) == INVALID, (T, kw)
    # the workspace of a long batch is that of a run of it
    assert size(16384, 4, 8, 256, 128, 0) == size(1 << 20, 4, 8, 256, 128, 0) > size(8000, 4, 8, 256, 128, 0)


def test_torch_operators():
    from my_int4 import _C
    from wush_int4_kernel_amd import _C as C2
    for op in ("quant_fp8_block", "fp8_gemm", "fp8_linear", "moe_route", "fp8_experts"):
        assert getattr(_C, op) is getattr(C2, op)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w, s = plain.weights(torch.Generator().manual_seed(0), 8, 128)
    e = torch.zeros(2, 256, 128).to(plain.E4M3), torch.ones(2, 2, 1), torch.zeros(2, 128, 128).to(plain.E4M3), torch.ones(2, 1, 1)
    for call in (lambda: _C.quant_fp8_block(x), lambda: _C.fp8_linear(x, w, s), lambda: _C.fp8_gemm(w, s, w, s), lambda: _C.moe_route(x, 2),
                 lambda: _C.fp8_experts(x, torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32), *e)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (300, 272), (3, 256, 144)])
def test_quant_weight(shape):
    from my_int4.decoder import quant_weight_fp8
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * 0.1
    w[..., 0, :] = 0
    q, s = quant_weight_fp8(w)
    N, K = shape[-2:]
    assert q.dtype == plain.E4M3 and q.shape == w.shape and q.is_contiguous() and s.shape == (*shape[:-2], -(-N // 128), -(-K // 128))
    v = q.double() * plain.spread(s, N, K)
    # half a step: 2^-4 of the value, or of the smallest normal's step, 2^-10 of a scale
    assert bool(((v - w.double()).abs() <= 2.0 ** -4 * 1.0001 * w.double().abs() + 2.0 ** -10 * 1.0001 * plain.spread(s, N, K)).all())
    assert bool(((q.float().abs().flatten(-2).amax(-1) == 448) | (w.abs().flatten(-2).amax(-1) == 0)).all())
    zero, one = quant_weight_fp8(torch.zeros(130, 16))
    assert not bool(zero.float().any()) and bool((one > 0).all())


def test_oracle_rounds_as_torch_does():
    v = torch.cat((torch.linspace(-460, 460, 20001), torch.linspace(-0.05, 0.05, 4001), torch.tensor([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, -0.0])))
    assert torch.equal(plain.nearest(v.double()).float(), v.to(plain.E4M3).float())
    q = torch.tensor([[256.0, 4.0, 8.0, 1.0, -2.0, 0, 0, 0]], dtype=torch.float64)
    w = torch.tensor([[256.0, 1.0, 1.0, 256.0, 256.0, 0, 0, 0]], dtype=torch.float64)
    # 2^16 and what of 4, 8, 256 and -512 is above 2^3
    assert float(plain.matrix_sums(q, w)) == 65536 + 0 + 8 + 256 - 512
