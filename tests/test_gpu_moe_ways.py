"""The experts' layers on each way that the plan chooses between, against what that way computes: which products the
matrix instruction cuts, and what an expert's rows are held in."""
from __future__ import annotations

import math

import pytest
import torch

import _fp8 as plain
from test_gpu_moe import case, gen

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]

# (gate and up products cut, down products cut, half a unit of the rows' type)
EXACT, DOWN, HALF = (False, False, 0.0), (False, True, 0.0), (False, True, 2.0 ** -11)
ALL = (True, True, 2.0 ** -11)                                   # no way's: what the e4m3 instruction would make of the hidden codes


def plan_of(T, k, E, H, I, dtype):
    from wush_int4_kernel_amd import capi
    return capi.moe_experts_fp8_plan(T, k, E, H, I, capi.DTYPE_BF16 if dtype == torch.bfloat16 else capi.DTYPE_F16)


def model_of(plan, dtype):
    from wush_int4_kernel_amd import capi
    if plan[0] == capi.MOE_DOT:
        return EXACT
    return HALF if plan[0] == capi.MOE_FUSED and dtype == torch.bfloat16 else DOWN


def spread_of(dtype, model, codes):
    """The relative error in root mean square that roundings leave against the way's own products.

    y: half a unit evenly spread, UNIT / sqrt 3 of a value at most; fp16 rows likewise.  Hidden codes that fall to another
    side of a half than the model's: a hidden value is off by up to 2^-21 (silu), 2^-22 (the factor) and, for each of gate
    and up, some 50 roundings of 2^-24 / sqrt 3, 2^-22: 2^-20 in all.  Codes are a step, 2^-4 to 2^-3 of the value, apart: one in 2^16
    turns at most, and is then a step, 2^-3.4 of the value in root mean square, off.  Of `codes` codes that many and four standard deviations
    more (and four more, for few) may turn; their values' squares are three times the mean at most, on average."""
    turned = (2.0 ** -16 * codes + 4 * (2.0 ** -16 * codes) ** 0.5 + 4) / codes
    return 1.1 * math.sqrt((plain.UNIT[dtype] ** 2 + model[2] ** 2) / 3 + 3 * turned * 2.0 ** -6.8)


def check_way(y, args, model):
    x, wts, ids = args[:3]
    ref, err = plain.experts(*args, *model)
    assert plain.off(y, ref, err, y.dtype) <= 1
    here = int(((ids >= 0) & (ids < args[3].shape[0])).sum())
    norm, got = float(ref.norm()), y.double()
    limit = spread_of(y.dtype, model, max(1, here * args[5].shape[2])) + 2.0 ** -25 * y.numel() ** 0.5 / norm
    assert float((got - ref).norm()) <= limit * norm
    # What the model leaves over (roundings, for the most part) has nothing to do with what sets the other models apart: on
    # the line from this model to another the outputs lie at 0, those of the other at 1, give or take |rest| / (sqrt n |line|).
    for other in (EXACT, DOWN, ALL):
        if other[:2] == model[:2]:
            continue
        line = plain.experts(*args, *other)[0] - ref
        far = float(line.norm())
        if 8 * limit * norm / y.numel() ** 0.5 < far:
            assert abs(float(((got - ref) * line).sum())) < 0.5 * far ** 2, other
    # and all of it: the roundings, and what this model is from the exact products
    exact = plain.experts(*args, *EXACT)[0]
    assert float((got - exact).norm()) <= limit * norm + float((ref - exact).norm())
    return float((ref - exact).norm()) / norm


def run(dev, dtype, shape, seed=0, away=0.0):
    from my_int4 import _C
    T, E, k, H, I = shape
    args = case(T + E + H + seed, T, E, k, H, I, dev, dtype, away)
    y = _C.fp8_experts(*args)
    assert torch.equal(y, _C.fp8_experts(*args))
    return y, args


# H up to 1024, 2048, 4096 and 8192, and I up to 1024, 2048 and 4096: a kernel each; more choices than wavefronts
DOT = [(1, 8, 2, 2048, 1408), (3, 64, 6, 2048, 1408), (2, 6, 3, 4096, 128), (1, 4, 2, 2720, 2176), (1, 3, 2, 8192, 256), (1, 4, 3, 6160, 4096),
       (1, 16, 12, 256, 1152), (40, 64, 6, 400, 384)]
# short last blocks of H, one and more blocks of I; what dot products do not take
ROWS = [(100, 64, 6, 400, 384), (90, 64, 6, 1040, 640), (20, 32, 8, 1040, 640), (64, 64, 8, 768, 128), (2, 8, 2, 512, 4352), (1, 8, 2, 256, 14336),
        (1, 8, 2, 8208, 256)]
# one tile for most experts, and several; one, two, three and more blocks of H and of I, H % 128 and H % 256 among them; more tiles of
# both products than the 256 workgroups that take them in turn (`many`)
ONCE = [(300, 32, 2, 640, 256), (120, 64, 8, 656, 1152), (400, 32, 2, 656, 384), (300, 60, 3, 1040, 640)]
FUSED = [(64, (200, 8, 2, 640, 256), False), (64, (1100, 64, 2, 1040, 640), True), (64, (1150, 64, 2, 272, 2560), False),
         (64, (1200, 64, 2, 2064, 384), False), (64, (1100, 64, 2, 128, 640), False), (128, (3000, 16, 2, 1296, 640), True),
         (128, (2500, 16, 2, 2064, 128), False), (128, (2500, 16, 2, 2064, 256), False), (128, (900, 16, 2, 112, 2560), False),
         (128, (2200, 20, 2, 272, 2560), False), (128, (2200, 20, 2, 1040, 1664), False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", DOT)
def test_dot_products(dev, shape, dtype):
    from wush_int4_kernel_amd import capi
    T, E, k, H, I = shape
    assert plan_of(T, k, E, H, I, dtype)[0] == capi.MOE_DOT
    check_way(*run(dev, dtype, shape), EXACT)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROWS)
def test_rows(dev, shape, dtype):
    from wush_int4_kernel_amd import capi
    T, E, k, H, I = shape
    assert plan_of(T, k, E, H, I, dtype)[:2] == (capi.MOE_ROWS, 32)
    check_way(*run(dev, dtype, shape), DOWN)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ONCE)
def test_fused_once(dev, shape, dtype):
    from wush_int4_kernel_amd import capi
    T, E, k, H, I = shape
    plan = plan_of(T, k, E, H, I, dtype)
    assert plan == (capi.MOE_FUSED, 64, 1, T)
    check_way(*run(dev, dtype, shape), model_of(plan, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,shape,many", FUSED)
def test_fused(dev, rows, shape, many, dtype):
    from wush_int4_kernel_amd import capi
    T, E, k, H, I = shape
    plan = plan_of(T, k, E, H, I, dtype)
    assert plan == (capi.MOE_FUSED, rows, 0, T)
    y, args = run(dev, dtype, shape)
    tiles = int(((torch.bincount(args[2].flatten().long(), minlength=E) + rows - 1) // rows).sum())
    if many:
        assert tiles * (I // 128) > 256 and tiles * -(-H // 256) > 256
    check_way(y, args, model_of(plan, dtype))


@pytest.mark.parametrize("shape", [(52, 64, 8, 400, 1408), (8, 8, 2, 256, 14336)])
def test_few_rows_of_many_columns(dev, shape):
    # few rows an expert, but workgroups enough for the gate and up projections
    from wush_int4_kernel_amd import capi
    T, E, k, H, I = shape
    for dtype in DTYPES:
        plan = plan_of(T, k, E, H, I, dtype)
        assert plan[:3] == (capi.MOE_FUSED, 64, 1)
        check_way(*run(dev, dtype, shape), model_of(plan, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_s_batch(dev, dtype):
    """A decode step's batch over many wide experts, half of the choices elsewhere."""
    shape = (51, 128, 8, 1024, 1024)
    T, E, k, H, I = shape
    plan = plan_of(T, k, E, H, I, dtype)
    check_way(*run(dev, dtype, shape, away=0.5), model_of(plan, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [ONCE[1], FUSED[1][1], FUSED[5][1], ROWS[1], DOT[1]])
def test_non_finite_tokens_stay_alone(dev, shape, dtype):
    from my_int4 import _C
    y, args = run(dev, dtype, shape, seed=1)
    bad = torch.arange(shape[0], device=dev) % 9 == 1
    args[0][bad, shape[3] - 1] = math.inf
    got = _C.fp8_experts(*args)
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], y[~bad])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(300, 60, 8, 2048, 1408), (700, 16, 3, 1040, 1280), (100, 64, 6, 400, 384), (51, 128, 8, 2048, 512)])
def test_outlier_channels(dev, shape, dtype):
    """Activations with some channels twenty times the others, next to whose products the matrix instruction cuts the others': the
    hidden codes are those of exact sums all the same.  Against 64 bits: the roundings, and the down projection's cut, 7 of 8
    products by 2^-13 of the largest at most, sqrt(7 / 3) 2^-13 of their root sum of squares."""
    from my_int4 import _C
    T, E, k, H, I = shape
    args = case(T + H, T, E, k, H, I, dev, torch.float32)
    args[0][:, torch.randperm(H, generator=gen(5))[:H // 100].to(dev)] *= 20
    args[0] = args[0].to(dtype)
    y = _C.fp8_experts(*args)
    model = model_of(plan_of(T, k, E, H, I, dtype), dtype)
    check_way(y, args, model)
    exact = plain.experts(*args, *EXACT)[0]
    limit = math.hypot(spread_of(dtype, model, T * k * I), 2.0 ** -13 * (7 / 3) ** 0.5)
    assert float((y.double() - exact).norm() / exact.norm()) <= limit
