"""e4m3 linear layers on the GPU: codes and scales equal the formulas' bit for
bit; products are within the rounding bounds of fp32 sums."""
from __future__ import annotations

import math

import pytest
import torch

import _fp8 as plain

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def acts(g, *shape, dtype=torch.bfloat16):
    x = torch.randn(*shape, generator=g)
    x[..., torch.randint(shape[-1], (max(1, shape[-1] // 100),), generator=g)] *= 20
    return x.to(dtype)


def check(y, q, s, w, ws, shape):
    """Within the bound of what the kernel of that shape computes, and near the exact product: cut products are off by
    at most 2^-13 of a group's largest, 7 of 8 of them, rms 2^-13 / sqrt(3) each, and the largest's square is
    part of the products' sum of squares."""
    from wush_int4_kernel_amd import capi
    ref, err = plain.product(q, s, w, ws)
    norm = float((y.double() - ref).norm() / ref.norm())
    assert norm <= 1.1 * math.hypot(plain.UNIT[y.dtype] / 3 ** 0.5, 2.0 ** -13 * (7 / 3) ** 0.5) + 2.0 ** -25 * y.numel() ** 0.5 / float(ref.norm())
    if capi.gemm_fp8_plan(*shape)[0] == capi.FP8_TILES:
        ref, err = plain.product(q, s, w, ws, matrix=True)
    assert plain.off(y, ref, err, y.dtype) <= 1


def same_quant(q, s, x):
    eq, es = plain.quant(x.reshape(-1, x.shape[-1]))
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.dtype == torch.float32
    assert torch.equal(q.cpu().float().reshape(eq.shape), eq.float())
    assert torch.equal(torch.nan_to_num(s.cpu().t(), nan=-1.0), torch.nan_to_num(es.float(), nan=-1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,K", [(1, 16), (3, 48), (5, 4096), (15, 144), (16, 128), (17, 2064), (130, 2064), (2, 16400), (1, 131056)])
def test_quant_bits(dev, dtype, rows, K):
    from my_int4 import _C
    x = acts(gen(rows + K), rows, K, dtype=dtype)
    same_quant(*_C.quant_fp8_block(x.to(dev)), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_special_blocks(dev, dtype):
    from my_int4 import _C
    g = gen(1)
    for rows in (12, 20):
        x = acts(g, rows, 272, dtype=dtype)
        x[0] = 0
        x[1, 5] = math.inf
        x[2, 200] = -math.inf
        x[3, 271] = math.nan
        x[4] = torch.finfo(dtype).tiny * 2.0 ** -3              # subnormal
        x[5] = torch.finfo(dtype).max
        x[6] = 0
        x[6, 7] = -1.0
        x[7] = torch.arange(272).to(dtype) * 0.5                # many halves between codes
        x[8] = (torch.arange(272) - 136).to(dtype) * torch.finfo(dtype).smallest_normal
        x[9] = (torch.randint(1, 256, (272,), generator=g) * 2.0 ** -8).to(dtype)
        x[10] = torch.finfo(dtype).smallest_normal * 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -24
        q, s = _C.quant_fp8_block(x.to(dev))
        same_quant(q, s, x)
        bad = torch.isnan(s.cpu()).t()
        assert bad[1].tolist() == [True, False, False] and bad[2].tolist() == [False, True, False]
        assert bad[3].tolist() == [False, False, True] and int(bad.sum()) == 3
        w, ws = plain.weights(g, 40, 272)
        y = _C.fp8_linear(x.to(dev), w.to(dev), ws.to(dev)).cpu()
        assert torch.isnan(y[1:4]).all() and torch.equal(y[0], torch.zeros_like(y[0]))
        ok = torch.tensor([4, 6, 7, 9])
        check(y[ok], *(t[ok] for t in plain.quant(x)), w, ws, (rows, 40, 272))


# one row to several tiles; widths and depths that end inside every tile and block
SHAPES = [(1, 1, 16), (1, 5, 128), (1, 4096, 1024), (1, 333, 8192), (2, 1000, 272), (3, 300, 2048), (4, 96, 4096), (5, 31, 80),
          (8, 2048, 2048), (13, 130, 1088), (16, 64, 256), (17, 65, 4160), (31, 515, 128), (33, 1024, 512), (48, 77, 2048),
          (64, 640, 1024), (65, 257, 320), (100, 1111, 192), (128, 129, 128), (129, 514, 2112), (200, 384, 4096),
          (255, 100, 960), (257, 700, 1024), (300, 2050, 128), (512, 512, 512), (700, 1027, 576), (1030, 520, 256),
          (40, 4000, 144), (300, 300, 48), (2100, 2600, 400)]


def check_product(_C, dev, M, N, K, dtypes=DTYPES):
    g = gen(M * 7 + N * 3 + K)
    xq = (torch.randn(M, K, generator=g) * 100).clamp(-448, 448).to(plain.E4M3).to(dev)
    xs = torch.exp(torch.randn(-(-K // 128), M, generator=g)).to(dev) * 2.0 ** -10
    w, ws = plain.weights(g, N, K, dev=dev)
    for dtype in dtypes:
        y = _C.fp8_gemm(xq, xs, w, ws, dtype=dtype)
        assert y.shape == (M, N) and y.dtype == dtype
        check(y, xq.float().double(), xs.t().double(), w, ws, (M, N, K))
        assert torch.equal(y, _C.fp8_gemm(xq, xs, w, ws, dtype=dtype))


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(dev, M, N, K):
    from my_int4 import _C
    check_product(_C, dev, M, N, K)


@pytest.mark.parametrize("M,N,K", [(2050, 8200, 128), (4096, 8192, 384), (2049, 12296, 272), (1900, 20480, 1040), (5000, 4104, 512),
                                   (4097, 4100, 256), (3000, 3333, 144)])
def test_more_tiles_than_workgroups(dev, M, N, K):
    # tiles one after another in a workgroup, of one block of K on; rows in every tile
    from my_int4 import _C
    g = gen(M + N + K)
    xq = (torch.randn(M, K, generator=g) * 100).clamp(-448, 448).to(plain.E4M3).to(dev)
    xs = torch.exp(torch.randn(-(-K // 128), M, generator=g)).to(dev) * 2.0 ** -10
    w, ws = plain.weights(g, N, K, dev=dev)
    rows = torch.cat((torch.arange(0, M, 61), torch.tensor([M - 2, M - 1]))).to(dev)
    for dtype in DTYPES:
        y = _C.fp8_gemm(xq, xs, w, ws, dtype=dtype)
        check(y[rows], xq[rows].float().double(), xs.t()[rows].double(), w, ws, (M, N, K))
        assert torch.equal(y, _C.fp8_gemm(xq, xs, w, ws, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 70, 96), (1, 4096, 4096), (3, 520, 1024), (7, 33, 16), (12, 515, 8192), (66, 200, 640),
                                   (260, 520, 1024)])
def test_linear(dev, dtype, M, N, K):
    from my_int4 import _C
    g = gen(M + N + K)
    x = acts(g, M, K, dtype=dtype)
    w, ws = plain.weights(g, N, K, dev=dev)
    y = _C.fp8_linear(x.to(dev), w, ws)
    check(y, *plain.quant(x.to(dev)), w, ws, (M, N, K))


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_layouts(dev, M):
    # leading dimensions, rows apart, misaligned and transposed inputs: the same bits
    from my_int4 import _C
    g = gen(M)
    K, N = 272, 150
    x = acts(g, M, K).to(dev)
    w, ws = plain.weights(g, N, K, dev=dev)
    y = _C.fp8_linear(x, w, ws)
    wide = torch.full((M, K + 40), math.nan, dtype=x.dtype, device=dev)
    for at in (0, 8, 3):
        wide[:, at:at + K] = x
        assert torch.equal(_C.fp8_linear(wide[:, at:at + K], w, ws), y)
        assert torch.equal(_C.quant_fp8_block(wide[:, at:at + K])[0].view(torch.uint8), _C.quant_fp8_block(x)[0].view(torch.uint8))
    assert torch.equal(_C.fp8_linear(x.t().contiguous().t(), w, ws), y)
    assert torch.equal(_C.fp8_linear(x.view(M, 1, K), w, ws), y.view(M, 1, N))
    q, s = _C.quant_fp8_block(x.view(1, M, K))
    assert q.shape == (1, M, K) and s.shape == (3, M)
    assert torch.equal(_C.fp8_gemm(q, s, w, ws), y.view(1, M, N))
    one = _C.fp8_linear(x[:1], w, ws)
    assert torch.equal(_C.fp8_linear(x[0], w, ws), one[0])
    many = _C.fp8_linear(x[:1].expand(M, K), w, ws)               # rows with stride 0
    assert torch.equal(many, many[:1].expand(M, N)) and torch.equal(many, _C.fp8_linear(x[:1].expand(M, K).contiguous(), w, ws))


def test_empty(dev):
    from my_int4 import _C
    w, ws = plain.weights(gen(0), 8, 64, dev=dev)
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device=dev)
    assert _C.fp8_linear(x[:0], w, ws).shape == (0, 8)
    assert _C.fp8_linear(x, w[:0], ws[:0]).shape == (3, 0)
    q, s = _C.quant_fp8_block(x[:0].view(2, 0, 64))
    assert q.shape == (2, 0, 64) and s.shape == (1, 0)


def test_nan_code_stays_in_its_column(dev):
    from my_int4 import _C
    g = gen(5)
    for M in (1, 30, 300):
        x = acts(g, M, 400).to(dev)
        w, ws = plain.weights(g, 130, 400, dev=dev)
        clean = _C.fp8_linear(x, w, ws)
        w.view(torch.uint8)[7, 399] = 0x7f
        ws[1, 0] = math.nan
        y = _C.fp8_linear(x, w, ws)
        assert torch.isnan(y[:, 7]).all() and torch.isnan(y[:, 128:]).all()
        keep = [n for n in range(128) if n != 7]
        assert torch.equal(y[:, keep], clean[:, keep])


@pytest.mark.parametrize("M,N,K", [(640, 32768, 256), (300, 65536, 144), (60, 131072, 128)])
def test_non_finite_rows_and_scales_stay_alone_from_tile_to_tile(dev, M, N, K):
    # more tiles than workgroups, one after another
    from my_int4 import _C
    g = gen(31)
    x = acts(g, M, K).to(dev)
    w, ws = plain.weights(g, N, K, dev=dev)
    clean = _C.fp8_linear(x, w, ws)
    bad = x.clone()
    bad[::7, 3] = math.inf
    y = _C.fp8_linear(bad, w, ws)
    keep = torch.ones(M, dtype=torch.bool, device=dev)
    keep[::7] = False
    assert torch.isnan(y[~keep]).all()
    assert torch.equal(y[keep], clean[keep])
    ws[::5, 0] = math.nan
    y = _C.fp8_linear(x, w, ws)
    cols = (torch.arange(N, device=dev) // 128) % 5 == 0
    assert torch.isnan(y[:, cols]).all()
    assert torch.equal(y[:, ~cols], clean[:, ~cols])


def test_graph_and_stream(dev):
    from my_int4 import _C
    g = gen(8)
    for M, N, K in [(1, 256, 512), (20, 520, 1024), (260, 512, 1024)]:
        x = acts(g, M, K).to(dev)
        w, ws = plain.weights(g, N, K, dev=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y1 = _C.fp8_linear(x, w, ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _C.fp8_linear(x, w, ws)
        for i in range(3):
            if i:
                x.copy_(acts(g, M, K).to(dev))
            expect = _C.fp8_linear(x, w, ws)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, expect)
            if i == 0:
                assert torch.equal(y1, expect)


def test_refusals(dev):
    from my_int4 import _C
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=dev)
    w, ws = plain.weights(gen(0), 8, 64, dev=dev)
    q, s = _C.quant_fp8_block(x)
    bad = [
        ("bf16 or fp16", lambda: _C.quant_fp8_block(x.float())),
        ("multiple of 16", lambda: _C.quant_fp8_block(x[:, :40])),
        ("multiple of 16", lambda: _C.quant_fp8_block(torch.zeros(1, 131072, dtype=torch.bfloat16, device=dev))),
        ("K mismatch", lambda: _C.fp8_linear(x[:, :48], w, ws)),
        ("one scale per 128", lambda: _C.fp8_linear(x, w, ws.expand(2, 1).contiguous())),
        ("float8_e4m3fn", lambda: _C.fp8_linear(x, w.float(), ws)),
        ("float8_e4m3fn", lambda: _C.fp8_linear(x, w.t().contiguous().t(), ws)),
        ("fp32", lambda: _C.fp8_linear(x, w, ws.half())),
        ("2D", lambda: _C.fp8_linear(x, w[0], ws)),
        ("CUDA", lambda: _C.fp8_linear(x.cpu(), w, ws)),
        ("CUDA", lambda: _C.fp8_linear(x, w.cpu(), ws)),
        ("xs must be", lambda: _C.fp8_gemm(q, s[:, :1].contiguous(), w, ws)),
        ("float8_e4m3fn", lambda: _C.fp8_gemm(x, s, w, ws)),
        ("bf16 or fp16", lambda: _C.fp8_gemm(q, s, w, ws, dtype=torch.float32)),
    ]
    for text, call in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
