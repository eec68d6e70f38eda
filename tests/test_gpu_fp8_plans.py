"""e4m3 products on every tile, split and dot product that the plan chooses between: each shape is here for a kernel,
and the plan query has to name that one."""
from __future__ import annotations

import math

import pytest
import torch

import _fp8 as plain
from test_gpu_fp8 import DTYPES, check

pytestmark = pytest.mark.gpu
WORKGROUPS = 256                                                 # of the kernels that take tiles one after another


def inputs(M, N, K, dev):
    g = torch.Generator(device=dev).manual_seed(M * 7 + N * 3 + K)

    def normal(*n):
        return torch.randn(*n, generator=g, device=dev)

    xq = (normal(M, K) * 100).clamp(-448, 448).to(plain.E4M3)
    xs = torch.exp(normal(-(-K // 128), M)) * 2.0 ** -10
    w = ((normal(N, K) * torch.exp(normal(N, 1))).clamp(-3, 3) * 149).to(plain.E4M3)
    return xq, xs, w, torch.exp(0.5 * normal(-(-N // 128), -(-K // 128))) * 2.0 ** -12


def close(y, q, s, w, ws, shape):
    """check(), whose bound of the norm takes roundings to be spread evenly, 3^-0.5 of half a unit in root mean square.  A few
    outputs may all be off by nearly half a unit (three roundings of 0.8 of it are 1.4 of that root mean square), so
    that they have the bound of each output only."""
    if y.numel() >= 100:
        return check(y, q, s, w, ws, shape)
    ref, err = plain.product(q, s, w, ws)
    assert plain.off(y, ref, err, y.dtype) <= 1


def check_product(dev, M, N, K, dtypes=DTYPES):
    from my_int4 import _C
    xq, xs, w, ws = inputs(M, N, K, dev)
    for dtype in dtypes:
        y = _C.fp8_gemm(xq, xs, w, ws, dtype=dtype)
        close(y, xq.float().double(), xs.t().double(), w, ws, (M, N, K))
        assert torch.equal(y, _C.fp8_gemm(xq, xs, w, ws, dtype=dtype))


# More tiles than workgroups; one, two, three and more blocks of K, the last one whole or short; columns that end inside a
# tile; rows that leave a tile's second half of wavefronts nothing (M % rows <= rows / 2), or something.
RUNS = {64: [(5, 65544, 112), (12, 65544, 128), (33, 65544, 112), (12, 65544, 144), (33, 65544, 256), (63, 65544, 144), (5, 65544, 384),
             (12, 200008, 272), (33, 65544, 272), (63, 65544, 512), (33, 65544, 400), (40, 65544, 1040), (40, 131080, 640)],
        128: [(70, 65544, 112), (100, 65544, 128), (90, 131080, 112), (130, 131080, 144), (70, 65544, 256), (130, 131080, 272), (90, 65544, 384),
              (130, 131080, 400), (70, 65544, 512), (100, 65544, 640), (90, 65544, 1040)]}


@pytest.mark.parametrize("rows,shape", [(r, s) for r in RUNS for s in RUNS[r]])
def test_tiles_one_after_another(dev, rows, shape):
    from wush_int4_kernel_amd import capi
    M, N, K = shape
    assert capi.gemm_fp8_plan(M, N, K) == (capi.FP8_TILES, rows, 256, 1)
    assert -(-M // rows) * -(-N // 256) > WORKGROUPS and N % 256
    check_product(dev, M, N, K)


@pytest.mark.parametrize("rows,shape", [(64, (12, 65544, 384)), (64, (40, 65544, 1040)), (64, (33, 65544, 112)), (128, (100, 65544, 640)),
                                        (128, (130, 131080, 144)), (128, (90, 65544, 1040))])
def test_non_finite_from_tile_to_tile(dev, rows, shape):
    from my_int4 import _C
    from wush_int4_kernel_amd import capi
    M, N, K = shape
    assert capi.gemm_fp8_plan(M, N, K) == (capi.FP8_TILES, rows, 256, 1)
    xq, xs, w, ws = inputs(M, N, K, dev)
    clean = _C.fp8_gemm(xq, xs, w, ws)
    bad = xs.clone()
    bad[-1, ::7] = math.nan
    y = _C.fp8_gemm(xq, bad, w, ws)
    of = torch.arange(M, device=dev) % 7 == 0
    assert torch.isnan(y[of]).all() and torch.equal(y[~of], clean[~of])
    ws[::5, -1] = math.nan
    y = _C.fp8_gemm(xq, xs, w, ws)
    of = (torch.arange(N, device=dev) // 128) % 5 == 0
    assert torch.isnan(y[:, of]).all() and torch.equal(y[:, ~of], clean[:, ~of])


# One tile a workgroup, in one pass over K and in slices of it; odd widths and depths among them
ONE = {(128, 128): [(70, 16392, 112), (90, 16393, 144), (203, 10000, 272), (100, 16390, 640), (203, 10001, 1040)],
       (64, 128): [(33, 16392, 112), (40, 16393, 272), (63, 16390, 400), (50, 16392, 1040), (400, 4104, 1024)],
       (32, 128): [(5, 16392, 128), (17, 16393, 144), (27, 16390, 1040), (5, 65544, 640), (500, 1032, 400)],
       (32, 64): [(5, 136, 112), (33, 520, 640), (27, 2055, 272), (170, 518, 1024)],
       (256, 256): [(170, 33000, 112), (400, 20487, 272), (400, 33000, 384)]}
SLICES = {(128, 128): [(100, 4104, 4096), (203, 8192, 8192), (400, 520, 8192), (203, 8185, 8208), (130, 4101, 8208)],
          (64, 128): [(33, 3000, 4096), (50, 10000, 4112), (40, 4101, 8208)],
          (32, 128): [(5, 4104, 4096), (5, 8200, 8208), (5, 4101, 4112)],
          (32, 64): [(5, 136, 2048), (40, 520, 4112), (13, 1031, 8208)]}


@pytest.mark.parametrize("tile,shape", [(t, s) for t in ONE for s in ONE[t]])
def test_tiles(dev, tile, shape):
    from wush_int4_kernel_amd import capi
    assert capi.gemm_fp8_plan(*shape) == (capi.FP8_TILES, *tile, 1)
    check_product(dev, *shape)


@pytest.mark.parametrize("tile,shape", [(t, s) for t in SLICES for s in SLICES[t]])
def test_slices(dev, tile, shape):
    from wush_int4_kernel_amd import capi
    plan = capi.gemm_fp8_plan(*shape)
    assert plan[:3] == (capi.FP8_TILES, *tile) and plan[3] > 1
    check_product(dev, *shape)


# Dot products: 8192 values of x in a workgroup's four wavefronts' registers, M C of 1024 each (M = 3 as 4): K in one slice a
# wavefront, two and four
DOTS = [(1, 8192), (1, 8208), (1, 16384), (1, 16400), (1, 32768), (2, 4096), (2, 4112), (2, 8192), (2, 8208), (2, 16384), (3, 2048), (3, 2064),
        (3, 4096), (3, 4112), (3, 8192), (4, 2048), (4, 2064), (4, 4096), (4, 4240), (4, 8192)]


@pytest.mark.parametrize("N", [3, 1000])
@pytest.mark.parametrize("M,K", DOTS)
def test_dot_products(dev, M, K, N):
    from my_int4 import _C
    from wush_int4_kernel_amd import capi
    assert capi.gemm_fp8_plan(M, N, K)[0] == capi.FP8_DOT
    check_product(dev, M, N, K)
    g = torch.Generator().manual_seed(M + K)
    w, ws = plain.weights(g, N, K, dev=dev)
    for dtype in DTYPES:
        x = torch.randn(M, K, generator=g).to(dtype).to(dev)
        close(_C.fp8_linear(x, w, ws), *plain.quant(x), w, ws, (M, N, K))


# Rows beyond a lane's registers go to the tiles, whose products are cut
@pytest.mark.parametrize("M,K", [(1, 32784), (2, 16400), (3, 8208), (4, 8320)])
def test_few_rows_of_great_depth(dev, M, K):
    from wush_int4_kernel_amd import capi
    assert capi.gemm_fp8_plan(M, 300, K)[0] == capi.FP8_TILES
    check_product(dev, M, 300, K)
