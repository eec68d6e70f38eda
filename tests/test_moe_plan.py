"""CPU checks of the experts' plan query: refusals, each way, and that it agrees with the workspace's size."""
from __future__ import annotations

import ctypes

import pytest

INVALID = 1
BF16, F16 = 0, 1


@pytest.fixture(scope="module")
def capi():
    from wush_int4_kernel_amd import capi as c
    c.load()
    return c


def test_refusals(capi):
    query, plan = capi.load().wush_moe_experts_fp8_plan, (ctypes.c_int32 * 4)()
    assert query(3, 2, 8, 256, 128, 0, plan) == 0
    assert query(3, 2, 8, 256, 128, 0, None) == INVALID
    for args in [(0, 2, 8, 256, 128, 0), (-1, 2, 8, 256, 128, 0), (3, 0, 8, 256, 128, 0), (3, 65, 8, 256, 128, 0), (3, 2, 0, 256, 128, 0),
                 (3, 2, 1025, 256, 128, 0), (3, 2, 8, 250, 128, 0), (3, 2, 8, 256, 100, 0), (3, 2, 8, 131072, 128, 0), (3, 2, 8, 256, 131072, 0),
                 (3, 2, 8, 256, 128, 2), (3, 2, 8, 256, 128, -1), ((1 << 26) + 1, 2, 8, 256, 128, 0)]:
        assert query(*args, plan) == INVALID, args


def test_ways(capi):
    plan = capi.moe_experts_fp8_plan
    for dtype in (BF16, F16):
        assert plan(1, 6, 64, 2048, 1408, dtype) == (capi.MOE_DOT, 0, 0, 1)
        # beyond what dot products take of H and I
        assert plan(1, 2, 8, 256, 14336, dtype)[0] == capi.MOE_ROWS == plan(1, 2, 8, 8208, 256, dtype)[0]
        assert plan(90, 6, 64, 1040, 640, dtype) == (capi.MOE_ROWS, 32, 1, 90)
        assert plan(400, 2, 32, 656, 384, dtype) == (capi.MOE_FUSED, 64, 1, 400)
        assert plan(1100, 2, 64, 1040, 640, dtype) == (capi.MOE_FUSED, 64, 0, 1100)
        assert plan(3000, 2, 16, 1296, 640, dtype) == (capi.MOE_FUSED, 128, 0, 3000)
        # few rows an expert of many columns
        assert plan(51, 8, 128, 4096, 1024, dtype) == (capi.MOE_FUSED, 64, 1, 51)


def test_runs(capi):
    # 65536 choices at once, fewer where rows are long: offsets of x and h stay below 2^31
    size = capi.load().wush_moe_experts_fp8_workspace_bytes
    for k, H, I, most in [(4, 128, 128, 16384), (1, 128, 128, 65536), (64, 128, 128, 1024), (1, 65536, 128, 32767), (8, 256, 65536, 4095)]:
        for T in (1000, 5000, 40000, 1 << 20):
            assert capi.moe_experts_fp8_plan(T, k, 4, H, I, BF16)[3] == min(T, most)
        assert size(70000, k, 4, H, I, BF16) == size(1 << 20, k, 4, H, I, BF16)


def test_another_way_s_products_are_told_apart():
    """The GPU tests' check refuses outputs whose gate and up products were cut."""
    import torch

    import _fp8 as plain
    from test_gpu_moe import case
    from test_gpu_moe_ways import ALL, DOWN, check_way
    args = case(3, 64, 4, 2, 512, 512, "cpu", torch.float16)
    y = plain.experts(*args, *ALL)[0].to(torch.float16)
    with pytest.raises(AssertionError):
        check_way(y, args, DOWN)
