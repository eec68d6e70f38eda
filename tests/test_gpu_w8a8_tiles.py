"""Every kernel and tile of the W8A8 product, bit for bit, each test with the plan
that its shape runs asserted, so that another plan cannot take it off its subject."""
from __future__ import annotations

import pytest
import torch

import _int8 as plain
from test_gpu_w8a8 import DTYPES, gen, same, weights

pytestmark = pytest.mark.gpu

# (M, N, K): (rows, columns, slices of K).  Rows and columns end inside a tile; K
# ends with a whole line of 128 codes or half of one; N is odd (stores of 2
# bytes), even (4) or a multiple of 8 (16); columns of tiles begin at different depths of K
TILES = {
    (5, 257, 4160): (32, 64, 7), (20, 4098, 4160): (32, 64, 3), (31, 1000, 576): (32, 64, 1),
    (31, 20001, 576): (32, 128, 1), (32, 24576, 512): (32, 128, 1), (13, 8200, 8256): (32, 128, 3), (5, 4098, 4096): (32, 128, 6),
    (33, 257, 4160): (64, 64, 7), (50, 1000, 1088): (64, 64, 1), (64, 514, 192): (64, 64, 1),
    (65, 8200, 576): (64, 128, 1), (100, 12290, 1088): (64, 128, 1), (33, 6001, 8256): (64, 128, 4), (33, 8200, 8192): (64, 128, 3),
    (65, 20001, 576): (128, 128, 1), (129, 12290, 1088): (128, 128, 1), (65, 24576, 512): (128, 128, 1),
    (65, 6001, 8256): (128, 128, 5), (65, 4096, 8192): (128, 128, 8),
    (257, 12290, 576): (256, 128, 1), (255, 20001, 512): (256, 128, 1), (500, 12288, 1024): (256, 128, 1),
    (129, 6001, 8256): (256, 128, 5), (129, 8192, 16448): (256, 128, 4),
    (257, 20001, 576): (256, 256, 1), (300, 28674, 512): (256, 256, 1), (511, 24576, 1088): (256, 256, 1),
    (129, 12290, 16448): (256, 256, 5),
}


def assert_plan(shape, kernel, *plan):
    from wush_int4_kernel_amd import capi
    assert capi.gemm_w8a8_plan(*shape) == (getattr(capi, kernel), *plan)


def operands(M, N, K):
    g = gen(M * 7 + N * 3 + K)
    xq = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int16).to(torch.int8)
    return xq, torch.exp(torch.randn(M, generator=g)), *weights(g, N, K)


@pytest.mark.parametrize("shape", TILES, ids=str)
def test_tiles(dev, shape):
    from my_int4 import _C
    assert_plan(shape, "W8A8_TILES", *TILES[shape])
    xq, xs, w, ws = operands(*shape)
    xs *= 2.0 ** -12
    on = [t.to(dev) for t in (xq, xs, w, ws)]
    sums = plain.product(xq, torch.ones_like(xs), w, torch.ones_like(ws), torch.float32)       # one rounding, as (float)sum
    for dtype in DTYPES:
        same(_C.w8a8_gemm(*on, dtype=dtype), (sums * xs[:, None] * ws).to(dtype))


@pytest.mark.parametrize("shape,columns", [((1, 4097, 1040), 4), ((2, 1001, 4096), 4), ((2, 16387, 4112), 8), ((3, 777, 1040), 4),
                                           ((3, 8197, 4096), 8), ((4, 32771, 4112), 16)], ids=str)
def test_dot_products(dev, shape, columns):
    # weight rows of a wavefront times four; widths that end inside one, a K behind whole 1024s
    from my_int4 import _C
    assert_plan(shape, "W8A8_DOT", shape[0], columns, 1)
    xq, xs, w, ws = operands(*shape)
    same(_C.w8a8_gemm(*(t.to(dev) for t in (xq, xs, w, ws)), dtype=torch.bfloat16), plain.product(xq, xs, w, ws, torch.bfloat16))


@pytest.mark.parametrize("shape", [(5, 33, 16), (17, 1001, 4112), (300, 514, 1040)], ids=str)
def test_streaming(dev, shape):
    from my_int4 import _C
    assert_plan(shape, "W8A8_STREAM", 16, 32, 1)
    xq, xs, w, ws = operands(*shape)
    same(_C.w8a8_gemm(*(t.to(dev) for t in (xq, xs, w, ws)), dtype=torch.bfloat16), plain.product(xq, xs, w, ws, torch.bfloat16))


@pytest.mark.parametrize("shape,plan", [((20, 48, 131008), (32, 64, 8)), ((300, 48, 131008), (64, 64, 8))], ids=str)
def test_largest_sum_on_tiles(dev, shape, plan):
    # the largest K that tiles take, every product 128 * 128: sums of 2^31 - 2^20
    from my_int4 import _C
    assert_plan(shape, "W8A8_TILES", *plan)
    M, N, K = shape
    xq = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    y = _C.w8a8_gemm(xq, torch.ones(M, device=dev), w, torch.ones(N, device=dev), dtype=torch.bfloat16)
    assert (y.float() == torch.tensor(16384.0 * K).bfloat16().float().item()).all()


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("shape", [(65, 8200, 576), (65, 4096, 8192), (257, 24576, 512)], ids=str)
def test_outputs_of_any_alignment(dev, shape, offset):
    # y 2, 4 or 8 bytes behind a multiple of 16, with and without slices; what lies around it stays
    from wush_int4_kernel_amd import capi
    lib = capi.load()
    M, N, K = shape
    xq, xs, w, ws = operands(*shape)
    xs *= 2.0 ** -12
    expect = plain.product(xq, xs, w, ws, torch.float16)
    on = [t.to(dev) for t in (xq, xs, w, ws)]
    need = lib.wush_gemm_w8a8_workspace_bytes(*shape)
    assert (need > 0) == (TILES.get(shape, (0, 0, 1))[2] > 1)
    work = torch.empty(need + 16, dtype=torch.uint8, device=dev)
    y = torch.full((M * N + 16,), 7.0, dtype=torch.float16, device=dev)
    assert lib.wush_gemm_w8a8(*[t.data_ptr() for t in on], y.data_ptr() + 2 * offset, capi.DTYPE_F16, *shape, work.data_ptr(), need,
                              torch.cuda.current_stream().cuda_stream) == 0
    same(y[offset:offset + M * N].view(M, N), expect)
    assert (y[:offset] == 7).all() and (y[offset + M * N:] == 7).all()


def test_streaming_more_rows_than_a_grid(dev):
    # 16 * 65535 rows are one launch
    from my_int4 import _C
    M, N, K = 16 * 65535 + 21, 5, 48
    assert_plan((M, N, K), "W8A8_STREAM", 16, 32, 1)
    xq, xs, w, ws = (t.to(dev) for t in operands(M, N, K))
    y = _C.w8a8_gemm(xq, xs, w, ws, dtype=torch.bfloat16)
    same(y, plain.product(xq.cpu(), xs.cpu(), w.cpu(), ws.cpu(), torch.bfloat16))
    x = xq.to(torch.bfloat16)                         # the layer too, whose rows are quantized in one launch
    q, s = _C.quant_int8_token(x)
    same(_C.w8a8_linear(x, w, ws), plain.product(q.cpu(), s.cpu(), w.cpu(), ws.cpu(), torch.bfloat16))


def test_quantizing_more_rows_than_a_launch(dev):
    # 2^21 rows are one launch, and 2^32 threads more than one can have: 2^26 rows of one wavefront
    from my_int4 import _C
    rows, K, piece = 2 ** 26 + 77, 16, 2 ** 21
    x = torch.empty(rows, K, dtype=torch.bfloat16, device=dev)
    x.copy_(torch.arange(rows, device=dev).remainder_(1009).sub_(504)[:, None])
    x += torch.arange(K, device=dev, dtype=torch.bfloat16)
    q, s = _C.quant_int8_token(x)
    for at in (0, piece - 50, 7 * piece - 50, 2 ** 25 - 50, 2 ** 26 - 50, rows - 100):
        eq, es = plain.quant_token(x[at:at + 100].cpu())
        same(q[at:at + 100], eq)
        same(s[at:at + 100], es)
