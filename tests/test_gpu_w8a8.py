"""W8A8 linear layers on the GPU: codes, scales and products equal the plain
form's bit for bit (the integer sum is exact, everything else a fixed
sequence of fp32 operations), at every size and whatever the strides."""
from __future__ import annotations

import math

import pytest
import torch

import _int8 as plain

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def acts(g, *shape, dtype=torch.bfloat16):
    x = torch.randn(*shape, generator=g)
    x[..., torch.randint(shape[-1], (max(1, shape[-1] // 100),), generator=g)] *= 20
    return x.to(dtype)


def weights(g, N, K):
    return (torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int16).to(torch.int8),
            torch.exp(torch.randn(N, generator=g)) * 0.01)


def same(a, b):
    a, b = a.cpu(), b.cpu()
    assert a.dtype == b.dtype and a.shape == b.shape
    nan = torch.isnan(b) if b.is_floating_point() else torch.zeros_like(b, dtype=torch.bool)
    assert torch.equal(a.isnan() if a.is_floating_point() else nan, nan)
    assert torch.equal(a[~nan], b[~nan]), (a[~nan] != b[~nan]).sum()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 16), (3, 48), (5, 4096), (130, 2064), (2, 16400), (1, 131056)])
def test_quant_bits(dev, dtype, rows, K):
    from my_int4 import _C
    x = acts(gen(rows + K), rows, K, dtype=dtype)
    q, s = _C.quant_int8_token(x.to(dev))
    eq, es = plain.quant_token(x)
    same(q, eq)
    same(s, es)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_special_rows(dev, dtype):
    from my_int4 import _C
    g = gen(1)
    x = acts(g, 9, 64, dtype=dtype)
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 63] = -math.inf
    x[3, 0] = math.nan
    x[4] = torch.finfo(dtype).tiny * 2.0 ** -3              # subnormal
    x[5] = torch.finfo(dtype).max
    x[6] = 0
    x[6, 7] = -1.0
    x[7] = torch.arange(64).to(dtype) * 0.5                 # halves of the largest: ties
    x[8] = (torch.arange(64) - 32).to(dtype) * torch.finfo(dtype).smallest_normal
    q, s = _C.quant_int8_token(x.to(dev))
    eq, es = plain.quant_token(x)
    same(q, eq)
    same(s, es)
    assert int(q.cpu()[0].abs().max()) == 0 and float(s.cpu()[0]) == 2.0 ** -126
    w, ws = weights(g, 40, 64)
    y = _C.w8a8_linear(x.to(dev), w.to(dev), ws.to(dev)).cpu()
    assert torch.isnan(y[1:4]).all() and torch.equal(y[0], torch.zeros_like(y[0]))
    same(y, plain.product(eq, es, w, ws, dtype))


# one row to several tiles; widths and depths that end inside every tile and step
SHAPES = [(1, 1, 16), (1, 5, 64), (1, 4096, 1024), (1, 333, 8192), (2, 1000, 272), (4, 96, 4096), (5, 31, 80),
          (8, 2048, 2048), (13, 130, 1088), (16, 64, 256), (17, 65, 4160), (31, 515, 128), (33, 1024, 512), (48, 77, 2048),
          (64, 640, 1024), (65, 257, 320), (100, 1111, 192), (128, 129, 64), (129, 514, 2112), (200, 384, 4096),
          (255, 100, 960), (257, 700, 1024), (300, 2050, 128), (512, 512, 512), (700, 1027, 576), (1030, 520, 256),
          (40, 4000, 144), (300, 300, 48)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_bits(dev, M, N, K):
    from my_int4 import _C
    g = gen(M * 7 + N * 3 + K)
    xq = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int16).to(torch.int8)
    xs = torch.exp(torch.randn(M, generator=g))
    w, ws = weights(g, N, K)
    for dtype in DTYPES:
        xs2 = xs * (2.0 ** -12 if dtype == torch.float16 else 1.0)
        y = _C.w8a8_gemm(xq.to(dev), xs2.to(dev), w.to(dev), ws.to(dev), dtype=dtype)
        same(y, plain.product(xq, xs2, w, ws, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 70, 96), (1, 4096, 4096), (3, 520, 1024), (7, 33, 16), (12, 515, 8192), (66, 200, 640),
                                   (260, 520, 1024)])
def test_linear_is_quant_and_product(dev, dtype, M, N, K):
    from my_int4 import _C
    g = gen(M + N + K)
    x = acts(g, M, K, dtype=dtype)
    w, ws = weights(g, N, K)
    y = _C.w8a8_linear(x.to(dev), w.to(dev), ws.to(dev))
    same(y, plain.product(*plain.quant_token(x), w, ws, dtype))


@pytest.mark.parametrize("M", [1, 20, 200])
def test_largest_sum_is_exact(dev, M):
    # every product 128 * 128: the sum reaches 16384 * 131056, just below 2^31
    from my_int4 import _C
    K = 131056
    xq = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((48, K), -128, dtype=torch.int8, device=dev)
    one = torch.ones(M, device=dev)
    y = _C.w8a8_gemm(xq, one, w, torch.ones(48, device=dev), dtype=torch.bfloat16)
    assert (y.float() == torch.tensor(16384.0 * K).bfloat16().float().item()).all()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_layouts(dev, M):
    # leading dimensions, rows apart, misaligned and transposed inputs: the same bits
    from my_int4 import _C
    g = gen(M)
    K, N = 256, 150
    x = acts(g, M, K)
    w, ws = (t.to(dev) for t in weights(g, N, K))
    y = _C.w8a8_linear(x.to(dev), w, ws)
    wide = torch.full((M, K + 40), math.nan, dtype=x.dtype, device=dev)
    for off in (0, 8, 3):
        wide[:, off:off + K] = x.to(dev)
        same(_C.w8a8_linear(wide[:, off:off + K], w, ws), y)
        same(_C.quant_int8_token(wide[:, off:off + K])[0], _C.quant_int8_token(x.to(dev))[0])
    same(_C.w8a8_linear(x.t().contiguous().to(dev).t(), w, ws), y)
    same(_C.w8a8_linear(x.to(dev).view(M, 1, K), w, ws), y.view(M, 1, N))
    q, s = _C.quant_int8_token(x.to(dev).view(1, M, K))
    assert q.shape == (1, M, K) and s.shape == (1, M)
    same(_C.w8a8_gemm(q, s, w, ws, dtype=torch.bfloat16), y.view(1, M, N))
    same(_C.w8a8_linear(x.to(dev)[0], w, ws), y[0])
    same(_C.w8a8_linear(x.to(dev)[:1].expand(M, K), w, ws), y[:1].expand(M, N))       # rows with stride 0


def test_empty(dev):
    from my_int4 import _C
    w, ws = (t.to(dev) for t in weights(gen(0), 8, 64))
    assert _C.w8a8_linear(torch.zeros(0, 64, dtype=torch.bfloat16, device=dev), w, ws).shape == (0, 8)
    assert _C.w8a8_linear(torch.zeros(3, 64, dtype=torch.bfloat16, device=dev), w[:0], ws[:0]).shape == (3, 0)
    q, s = _C.quant_int8_token(torch.zeros(2, 0, 64, dtype=torch.bfloat16, device=dev))
    assert q.shape == (2, 0, 64) and s.shape == (2, 0)


@pytest.mark.parametrize("M,N,K", [(1, 512, 2048), (30, 1024, 4096), (300, 512, 1024)])
def test_workspace_does_not_change_bits(dev, M, N, K):
    from wush_int4_kernel_amd import capi
    lib = capi.load()
    g = gen(3)
    xq = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int16).to(torch.int8)
    xs = torch.rand(M, generator=g) * 1e-3
    w, ws = weights(g, N, K)
    expect = plain.product(xq, xs, w, ws, torch.float16)
    d = [t.to(dev) for t in (xq, xs, w, ws)]
    st = torch.cuda.current_stream().cuda_stream
    need = lib.wush_gemm_w8a8_workspace_bytes(M, N, K)
    for size in {0, need, need + 4096}:
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
        y = torch.empty(M, N, dtype=torch.float16, device=dev)
        st_ = lib.wush_gemm_w8a8(*[t.data_ptr() for t in d], y.data_ptr(), capi.DTYPE_F16, M, N, K, work.data_ptr(), size, st)
        assert st_ == 0
        same(y, expect)


def test_graph_and_stream(dev):
    from my_int4 import _C
    g = gen(8)
    for M, N, K in [(1, 256, 512), (20, 520, 1024), (260, 512, 1024)]:
        x = acts(g, M, K).to(dev)
        w, ws = (t.to(dev) for t in weights(g, N, K))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y1 = _C.w8a8_linear(x, w, ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _C.w8a8_linear(x, w, ws)
        for i in range(3):
            if i:
                x.copy_(acts(g, M, K).to(dev))
            expect = _C.w8a8_linear(x, w, ws)
            graph.replay()
            torch.cuda.synchronize()
            same(y, expect)
            if i == 0:
                same(y1, expect)


def test_refusals(dev):
    from my_int4 import _C
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=dev)
    w, ws = torch.zeros(8, 64, dtype=torch.int8, device=dev), torch.ones(8, device=dev)
    q, s = _C.quant_int8_token(x)
    bad = [
        ("bf16 or fp16", lambda: _C.quant_int8_token(x.float())),
        ("multiple of 16", lambda: _C.quant_int8_token(x[:, :40])),
        ("multiple of 16", lambda: _C.quant_int8_token(torch.zeros(1, 131072, dtype=torch.bfloat16, device=dev))),
        ("K mismatch", lambda: _C.w8a8_linear(x[:, :48], w, ws)),
        ("one scale per row", lambda: _C.w8a8_linear(x, w, ws[:7])),
        ("int8", lambda: _C.w8a8_linear(x, w.float(), ws)),
        ("int8", lambda: _C.w8a8_linear(x, w.t().contiguous().t(), ws)),
        ("fp32", lambda: _C.w8a8_linear(x, w, ws.half())),
        ("2D", lambda: _C.w8a8_linear(x, w[0], ws)),
        ("CUDA", lambda: _C.w8a8_linear(x.cpu(), w, ws)),
        ("CUDA", lambda: _C.w8a8_linear(x, w.cpu(), ws)),
        ("one scale per row", lambda: _C.w8a8_gemm(q, s[:1], w, ws)),
        ("int8", lambda: _C.w8a8_gemm(x, s, w, ws)),
        ("bf16 or fp16", lambda: _C.w8a8_gemm(q, s, w, ws, dtype=torch.float32)),
        ("aligned", lambda: _C.w8a8_gemm(q, s, torch.zeros(8 * 64 + 8, dtype=torch.int8, device=dev)[8:].view(8, 64), ws)),
    ]
    for text, call in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
