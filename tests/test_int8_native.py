"""CPU checks of the 8-bit operators' host side: bad arguments are refused and
empty work succeeds before any device is touched; workspace sizes are host only;
the torch module exposes the operators and refuses CPU tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

INVALID = 1
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def capi():
    from wush_int4_kernel_amd import capi as c
    c.load()
    return c


def test_w8a8_arguments(capi):
    lib = capi.load()
    quant, gemm, linear = lib.wush_quant_int8_token, lib.wush_gemm_w8a8, lib.wush_linear_w8a8
    assert quant(None, 0, None, None, 0, 64, 64, None) == 0
    for args in [(None, 0, P(16), P(16), 1, 64, 64), (P(16), 2, P(16), P(16), 1, 64, 64), (P(8), 0, P(16), P(16), 1, 64, 64),
                 (P(16), 0, P(8), P(16), 1, 64, 64), (P(16), 0, P(16), P(16), 1, 40, 40), (P(16), 0, P(16), P(16), 1, 131072, 131072),
                 (P(16), 0, P(16), P(16), 2, 64, 60), (P(16), 0, P(16), P(16), 2, 64, 68), (P(16), 0, P(16), P(16), -1, 64, 64)]:
        assert quant(*args, None) == INVALID, args
    ok = [P(16)] * 5
    assert gemm(*[None] * 5, 0, 0, 8, 64, None, 0, None) == 0 and gemm(*[None] * 5, 0, 8, 0, 64, None, 0, None) == 0
    for args in [(*ok, 2, 1, 8, 64), (*ok, 0, 1, 8, 40), (*ok, 0, 1, 8, 131072), (*ok, 0, -1, 8, 64), (None, *ok[1:], 0, 1, 8, 64),
                 (P(8), *ok[1:], 0, 1, 8, 64), (*ok[:2], P(8), *ok[3:], 0, 1, 8, 64), (*ok[:4], P(1), 0, 1, 8, 64), (*ok, 0, 1, 8, 0)]:
        assert gemm(*args, None, 0, None) == INVALID, args
    assert linear(None, 64, None, None, None, 0, 0, 8, 64, None, 0, None) == 0
    need = lib.wush_linear_w8a8_workspace_bytes(4, 8, 64)
    assert need >= 4 * 64 + 16
    assert linear(P(16), 64, P(16), P(16), P(16), 0, 4, 8, 64, P(16), need - 1, None) == INVALID
    assert linear(P(16), 64, P(16), P(16), P(16), 0, 4, 8, 64, None, need, None) == INVALID
    assert linear(P(16), 60, P(16), P(16), P(16), 0, 4, 8, 64, P(16), need, None) == INVALID
    assert lib.wush_gemm_w8a8_workspace_bytes(0, 8, 64) == 0 == lib.wush_linear_w8a8_workspace_bytes(0, 8, 64)
    # int32 bound: codes of -128 on both sides
    assert 128 * 128 * 131056 < 2 ** 31 <= 128 * 128 * (131056 + 16)


def cache(capi, **kw):
    d = dict(k=16, v=16, k_scale=16, v_scale=16, pages=4, heads=2, page_size=16, head_dim=64)
    d.update(kw)
    return capi.Kv8Cache(**d)


BAD_CACHES = [dict(k=None), dict(v_scale=None), dict(k=8), dict(k_scale=2), dict(pages=0), dict(pages=1 << 31), dict(heads=0),
              dict(heads=1 << 16), dict(page_size=48), dict(page_size=8), dict(page_size=256), dict(head_dim=96), dict(head_dim=256)]


def test_kv8_arguments(capi):
    lib = capi.load()
    strides = (ctypes.c_int64 * 6)(256, 64, 256, 64, 256, 64)

    def append(c, q=P(16), k=P(16), v=P(16), dtype=0, st=strides, cs=P(16), positions=8, rot=64, table=P(16), ts=4, lens=P(16),
               cu=None, seqs=2, tokens=2, heads=4, out=P(16)):
        return lib.wush_kv8_append(q, k, v, dtype, st, cs, positions, rot, 0, ctypes.byref(c) if c else None, table, ts, lens, cu,
                                   seqs, tokens, heads, out, None)

    def attend(c, q=P(16), dtype=0, qt=256, qh=64, table=P(16), ts=4, lens=P(16), cu=None, seqs=2, tokens=2, heads=4, scale=0.1,
               window=0, cap=0.0, max_len=0, out=P(16), ws=None, wsb=0):
        return lib.wush_kv8_attention(q, dtype, qt, qh, ctypes.byref(c) if c else None, table, ts, lens, cu, seqs, tokens, heads,
                                      scale, window, cap, max_len, out, ws, wsb, None)

    def read(c, pages=P(16), n=1, dtype=0, k=P(16), v=P(16)):
        return lib.wush_kv8_read(ctypes.byref(c) if c else None, pages, n, dtype, k, v, None)

    for f in (append, attend, read):
        assert f(None) == INVALID
        for kw in BAD_CACHES:
            assert f(cache(capi, **kw)) == INVALID, (f, kw)
    c = cache(capi)
    assert append(c, seqs=0) == 0 and append(c, tokens=0) == 0 and attend(c, seqs=0) == 0 and attend(c, tokens=0) == 0
    assert read(c, n=0) == 0
    odd = (ctypes.c_int64 * 6)(256, 64, 256, 60, 256, 64)
    for kw in [dict(q=None), dict(k=P(8)), dict(v=None), dict(dtype=2), dict(st=odd), dict(st=None), dict(cs=None), dict(positions=0),
               dict(rot=24), dict(rot=80), dict(rot=-16), dict(table=None), dict(lens=None), dict(tokens=3), dict(seqs=-1), dict(ts=-1),
               dict(heads=-1), dict(out=None), dict(out=P(8)), dict(tokens=1 << 31, cu=P(16)), dict(heads=1 << 40)]:
        assert append(c, **kw) == INVALID, kw
    for kw in [dict(q=None), dict(q=P(8)), dict(dtype=2), dict(qt=60), dict(qh=4), dict(table=None), dict(lens=None), dict(tokens=3),
               dict(heads=3), dict(heads=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(cap=-1.0), dict(cap=float("nan")),
               dict(cap=float("inf")), dict(max_len=-1), dict(out=None), dict(seqs=-1), dict(ts=-1), dict(tokens=1 << 31, cu=P(16))]:
        assert attend(c, **kw) == INVALID, kw
    for kw in [dict(pages=None), dict(k=None), dict(v=P(8)), dict(dtype=2), dict(n=-1), dict(n=1 << 40)]:
        assert read(c, **kw) == INVALID, kw
    # a cache long enough to be split needs the workspace that it asks for
    need = lib.wush_kv8_attention_workspace_bytes(ctypes.byref(c), 2, 2, 0, 4, 4096, 0, 0)
    assert need > 0 and attend(c, ts=4096) == INVALID and attend(c, ts=4096, ws=P(16), wsb=need - 1) == INVALID
    assert attend(c, ts=4096, ws=P(8), wsb=need) == INVALID
    assert lib.wush_kv8_attention_workspace_bytes(ctypes.byref(c), 2, 2, 0, 4, 4096, 0, 64) == 0
    assert lib.wush_kv8_attention_workspace_bytes(ctypes.byref(cache(capi, head_dim=96)), 2, 2, 0, 4, 4096, 0, 0) == 0


def test_torch_operators():
    from my_int4 import _C
    from wush_int4_kernel_amd import _C as C2
    for op in ("quant_int8_token", "w8a8_gemm", "w8a8_linear", "kv8_append", "kv8_attention", "kv8_read"):
        assert getattr(_C, op) is getattr(C2, op)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, ws = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.quant_int8_token(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.w8a8_linear(x, w, ws)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.w8a8_gemm(w, ws, w, ws)
    k, s, i = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.ones(2, 1), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    v = k.transpose(2, 3).contiguous()
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.kv8_append(q, q, q, torch.zeros(1, 64), k, v, s, s, i[None], i)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.kv8_attention(q, k, v, s, s, i[None], i)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.kv8_read(k, v, s, s, i)


def test_window_wider_than_every_sequence_is_planned_as_none(capi):
    lib = capi.load()
    need = [lib.wush_kv8_attention_workspace_bytes(ctypes.byref(cache(capi, heads=8, head_dim=128)), 1, 1, 0, 64, 8192, w, 0)
            for w in (0, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 62)]
    assert need[0] > 0 and need == need[:1] * 6


def test_plan_queries(capi):
    lib = capi.load()
    plan = (ctypes.c_int32 * 4)()
    for args in [(0, 8, 64), (1, 0, 64), (1, 8, 40), (1, 8, 131072), (1, 8, 0)]:
        assert lib.wush_gemm_w8a8_plan(*args, 0, plan) == INVALID, args
    assert lib.wush_gemm_w8a8_plan(1, 8, 64, 0, None) == INVALID
    assert capi.gemm_w8a8_plan(4, 4096, 4096)[0] == capi.W8A8_DOT
    assert capi.gemm_w8a8_plan(5, 4096, 4112) == (capi.W8A8_STREAM, 16, 32, 1)
    kernel, _, _, slices = capi.gemm_w8a8_plan(13, 4096, 8192)
    assert kernel == capi.W8A8_TILES and slices > 1 and capi.gemm_w8a8_plan(13, 4096, 8192, 0)[3] == 1
    assert lib.wush_gemm_w8a8_workspace_bytes(13, 4096, 8192) == slices * 13 * 4096 * 4

    def attend(c, seqs=2, tokens=2, ragged=0, heads=4, ts=4, window=0, max_len=0, out=plan):
        return lib.wush_kv8_attention_plan(ctypes.byref(c), seqs, tokens, ragged, heads, ts, window, max_len, out)

    c = cache(capi)
    for kw in [dict(seqs=0), dict(tokens=0), dict(heads=3), dict(heads=0), dict(ts=-1), dict(window=-1), dict(max_len=-1), dict(out=None)]:
        assert attend(c, **kw) == INVALID, kw
    for kw in BAD_CACHES:
        assert attend(cache(capi, **kw)) == INVALID, kw
    assert attend(c) == 0 and list(plan) == [16, 1, 256, 0]
    rows, stretches, tokens, _ = capi.kv8_attention_plan(100, 8, 64, 128, 1, 1, False, 64, 2048)
    assert rows == 16 and stretches > 1 and (stretches - 1) * tokens < 2048 * 64 <= stretches * tokens
    need = lib.wush_kv8_attention_workspace_bytes(ctypes.byref(cache(capi, heads=8, page_size=64, head_dim=128)), 1, 1, 0, 64, 2048, 0, 0)
    assert need == 64 * stretches * (128 + 4) * 4
    # single tokens are taken by length where their sequences are long and fill the chip
    assert capi.kv8_attention_plan(100, 8, 64, 128, 64, 64, False, 64, 64)[3] == 32
    assert capi.kv8_attention_plan(100, 8, 64, 128, 64, 64, False, 64, 8)[3] == 0
