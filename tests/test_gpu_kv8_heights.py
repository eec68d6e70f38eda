"""Attention over the 8-bit cache in each form that the plan has for many query
rows, tiles of 128 and 256 rows, alone and with stretches joined.  Every test asserts the
plan that its shapes run, so that another plan cannot take it off its subject."""
from __future__ import annotations

import math

import pytest
import torch

import _int8 as plain
from test_gpu_kv8 import BF, HF, Batch, i32

pytestmark = pytest.mark.gpu

# rows of a tile, joined, and query heads, key/value heads, head_dim, page, lengths, new
# tokens; the last: a window narrow enough to hide tokens with which the plan is of the same kind
SHAPES = {
    "128-64": (128, False, 64, 4, 64, 16, [300, 64, 1, 65, 129, 40], [300, 64, 1, 65, 70, 0], 40),
    "128-128": (128, False, 28, 4, 128, 32, [300, 64, 1, 65, 129, 40], [300, 64, 1, 65, 70, 0], None),
    "128-64-joined": (128, True, 8, 2, 64, 64, [4100, 3500, 1, 4050], [400, 380, 1, 350], 2900),
    "128-128-joined": (128, True, 16, 2, 128, 16, [3100, 2500, 1, 3050, 65, 2900], [130, 80, 1, 100, 64, 160], 2000),
    "256-64": (256, False, 32, 2, 64, 32, [1420, 1300, 1, 700, 65, 1333], [1420, 1300, 1, 630, 64, 200], 1300),
    "256-128": (256, False, 64, 1, 128, 128, [420, 300, 1, 700, 65, 333], [420, 300, 1, 630, 64, 200], 600),
    "256-64-joined": (256, True, 16, 2, 64, 64, [3130, 3100, 3120, 3060, 65, 3090], [130, 100, 120, 90, 64, 90], None),
    "256-128-joined": (256, True, 16, 2, 128, 16, [3130, 3100, 3120, 3060, 65, 3090], [130, 100, 120, 90, 64, 90], 2500),
}


# the same for few rows, which have tests of their own
FEW = {
    "16": (16, False, 8, 2, 64, 16, [40, 9], [40, 9], None),
    "16-joined": (16, True, 8, 2, 128, 64, [3000, 700, 64], [5, 1, 9], None),
}


def batch(shape, dtype, seed=50, **kw):
    _, _, Hq, Hkv, D, page, lens, n, _ = {**SHAPES, **FEW}[shape]
    return Batch(seed, lens, n, Hq, Hkv, D, page, dtype, **kw)


def assert_plan(bt, shape, window=0):
    from wush_int4_kernel_amd import capi
    rows, stretches, _, _ = capi.kv8_attention_plan(bt.cache.k.shape[0], bt.Hkv, bt.page, bt.D, len(bt.lens), sum(bt.n), True,
                                                    bt.Hq, bt.table.shape[1], window, 0)
    assert (rows, stretches > 1) == {**SHAPES, **FEW}[shape][:2]


def reference(dev, bt, b, q, scale=None, window=0, cap=0.0):
    """plain.attention of sequence b's queries, in fp64 on the GPU."""
    k, v, seen = bt.cache.sequence(bt.pages[b], min(bt.lens[b], bt.table.shape[1] * bt.page))
    with torch.device(dev):
        return plain.attention(q, k.to(dev), v.to(dev), seen.to(dev), bt.lens[b] - bt.n[b],
                               bt.D ** -0.5 if scale is None else scale, window, cap)


def within(got, ref, bound):
    same_nan = torch.equal(torch.isnan(got), torch.isnan(ref))
    return same_nan and bool((torch.nan_to_num((got - ref).abs()) <= torch.nan_to_num(bound)).all())


def run(dev, bt, scale=None, window=0, cap=0.0):
    from my_int4 import _C
    table, lens, cu = bt.meta(dev)
    kw = {} if scale is None else {"scale": scale}
    return _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, lens, cu_q=cu, window=window, softcap=cap, **kw)


def check_attention(dev, bt, scale=None, window=0, cap=0.0, filled=True):
    if filled:
        bt.fill(bt.lens)
    out, q, at = run(dev, bt, scale, window, cap), bt.q.to(dev), 0
    for b, n in enumerate(bt.n):
        ref, A, E = reference(dev, bt, b, q[at:at + n], scale, window, cap)
        assert within(out[at:at + n].double(), ref, plain.attention_bound(ref, A, E, bt.dtype)), b
        at += n
    return out.cpu()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows(dev, shape, dtype):
    bt = batch(shape, dtype)
    assert_plan(bt, shape)
    out = check_attention(dev, bt)
    assert torch.equal(out, check_attention(dev, bt, filled=False))


@pytest.mark.parametrize("shape", [s for s in SHAPES if SHAPES[s][-1]])
def test_window(dev, shape):
    bt, window = batch(shape, HF, 51), SHAPES[shape][-1]
    assert_plan(bt, shape, window)
    check_attention(dev, bt, window=window)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", SHAPES)
def test_softcap(dev, shape, dtype):
    # scores on both sides of the cap, with a window where the plan stays
    bt, window = batch(shape, dtype, 52, size=4.0), (SHAPES[shape][-1] or 0) if dtype == BF else 0
    assert_plan(bt, shape, window)
    check_attention(dev, bt, cap=5.0 if dtype == BF else 30.0, window=window)


@pytest.mark.parametrize("shape", SHAPES)
def test_negative_scale(dev, shape):
    bt = batch(shape, HF, 53)
    assert_plan(bt, shape)
    check_attention(dev, bt, scale=-0.2)


@pytest.mark.parametrize("shape", SHAPES)
def test_missing_pages_are_not_seen(dev, shape):
    # the first page, pages in the middle, and the last of sequences; one sequence without any
    bt = batch(shape, BF, 54)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    last = bt.cache.k.shape[0]
    for b, p in ((0, 0), (0, 2), (1, len(bt.pages[1]) - 1), (3, len(bt.pages[3]) // 2)):
        bt.pages[b][p] = bt.table[b, p] = (-1, 2 ** 30, last)[p % 3]
    b = len(bt.pages) - 1
    bt.pages[b] = [-1] * len(bt.pages[b])
    bt.table[b] = -1
    out = check_attention(dev, bt, filled=False)
    at = sum(bt.n[:-1])
    assert torch.equal(out[at:], torch.zeros_like(out[at:]))


def small_weights(dev, bt, b, q):
    """What one sequence's outputs may lose with the bits of small weights, (n, Hq, D): a
    weight is p * v_scale, at least 2^12 for a row's largest, rounded to fp16, below
    2^-14 to multiples of 2^-24: off by 2^-25, times its code."""
    pages = [p for p in bt.pages[b] if 0 <= p < bt.cache.k.shape[0]]
    assert len(pages) * bt.page >= bt.lens[b]
    k, v, _ = bt.cache.sequence(bt.pages[b], bt.lens[b])
    vs = bt.cache.vs[pages].double().repeat_interleave(bt.page, 0)[:bt.lens[b]].to(dev)       # (L, Hkv)
    k, codes = k.to(dev), (v.to(dev) / vs[..., None]).abs().sum(0)                            # codes: (Hkv, D)
    pos = bt.lens[b] - bt.n[b] + torch.arange(bt.n[b], device=dev)[:, None]
    out = torch.empty(bt.n[b], bt.Hq, bt.D, dtype=torch.float64, device=dev)
    for hq in range(bt.Hq):
        h = hq // (bt.Hq // bt.Hkv)
        s = (q[:, hq].double() @ k[:, h].t()) * bt.D ** -0.5
        p = s.masked_fill(torch.arange(bt.lens[b], device=dev) > pos, -math.inf).softmax(-1)
        out[:, hq] = (p * vs[:, h]).amax(-1, keepdim=True) * codes[h] * 2.0 ** (-25 - 12)
    return out


@pytest.mark.parametrize("shape", SHAPES)
def test_scales_of_every_size(dev, shape):
    # pages of zeros, of tiny and of large values side by side, scores in the hundreds
    bt = batch(shape, BF, 55)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    for pages in bt.pages:
        for i, p in enumerate(pages):
            f = (1.0, 0.0, 2.0 ** -20, 2.0 ** 20, 2.0 ** -39)[i % 5]
            if f:
                bt.cache.vs[p] *= f
            else:
                bt.cache.v[p] = 0
                bt.cache.vs[p] = plain.FLOOR
            bt.cache.ks[p] *= (1.0, 40.0, 0.01)[i % 3]
    out, q, at = run(dev, bt), bt.q.to(dev), 0
    for b, n in enumerate(bt.n):
        ref, A, E = reference(dev, bt, b, q[at:at + n])
        assert within(out[at:at + n].double(), ref, plain.attention_bound(ref, A, E, BF) + small_weights(dev, bt, b, q[at:at + n])), b
        at += n


@pytest.mark.parametrize("shape", SHAPES)
def test_non_finite_values(dev, shape):
    # queries, and a page's scales, that are not finite: NaN for the rows that see them only
    from my_int4 import _C
    bt = batch(shape, BF, 56)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    bt.q[7, 1, 3] = math.nan
    bt.q[bt.n[0] + 20, 2, 9] = -math.inf
    b = 1                                             # the page of the sequence's 20th-last token on
    first = bt.lens[b] - 20
    page = bt.pages[b][first // bt.page]
    bt.cache.vs[page, 0] = math.nan
    bt.cache.ks[page, -1] = math.nan
    table, lens, cu = bt.meta(dev)
    out = _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, lens, cu_q=cu).float().cpu()
    expect = torch.zeros(sum(bt.n), bt.Hq, dtype=torch.bool)
    expect[7, 1] = expect[bt.n[0] + 20, 2] = True
    at = sum(bt.n[:b])
    pos = torch.arange(bt.n[b]) + bt.lens[b] - bt.n[b]
    sees = pos >= first // bt.page * bt.page
    G = bt.Hq // bt.Hkv
    expect[at:at + bt.n[b], :G] |= sees[:, None]
    expect[at:at + bt.n[b], -G:] |= sees[:, None]
    assert torch.equal(torch.isnan(out).all(-1), expect) and torch.equal(torch.isnan(out).any(-1), expect)


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_that_see_nothing(dev, shape):
    # tokens before position 0, a length of 0, tokens behind the table
    bt = batch(shape, HF, 57)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    bt.lens = [bt.n[0] // 2, 0] + bt.lens[2:]
    bt.lens[3] += 2 * bt.page
    out = check_attention(dev, bt, filled=False)
    none = bt.n[0] - bt.lens[0]
    assert torch.equal(out[:none], torch.zeros_like(out[:none])) and out[none].abs().sum() > 0
    assert not out[bt.n[0]:bt.n[0] + bt.n[1]].any()


def test_offsets_past_32_bits(dev):
    # tiles of 128 and 256 rows over the last pages of a cache of more than 2^31 codes a tensor
    from my_int4 import _C
    from wush_int4_kernel_amd import capi
    Hkv, D, page = 8, 128, 128
    pages = (2 ** 31 // (Hkv * D * page)) + 300
    k = torch.zeros(pages, Hkv, page, D, dtype=torch.int8, device=dev)
    v = torch.zeros(pages, Hkv, D, page, dtype=torch.int8, device=dev)
    ks, vs = (torch.full((pages, Hkv), math.nan, device=dev) for _ in range(2))
    for rows, Hq, room in ((128, 64, 0), (256, 32, 29)):
        bt = Batch(rows, [300], [300], Hq, Hkv, D, page, BF, spare=0)
        bt.fill([300])
        at = [pages - 1, 1, pages - 2]
        for t, c in zip((k, v, ks, vs), bt.cache.tensors()):
            t[at] = c[bt.pages[0]].to(dev)
        assert capi.kv8_attention_plan(pages, Hkv, page, D, 1, 300, True, Hq, 3 + room)[0] == rows
        table = i32([at + [-1] * room], dev)
        out = _C.kv8_attention(bt.q.to(dev), k, v, ks, vs, table, i32([300], dev), cu_q=i32([0, 300], dev))
        ref, A, E = reference(dev, bt, 0, bt.q.to(dev))
        assert within(out.double(), ref, plain.attention_bound(ref, A, E, BF))


@pytest.mark.parametrize("shape", ["16", "16-joined", "128-64", "128-128-joined", "256-128"])
@pytest.mark.parametrize("dtype,size", [(HF, 4e4), (BF, 1e6), (BF, 1e8), (BF, 4e8), (BF, 1e9), (BF, 1e18), (BF, 1e30), (BF, 1e-30), (BF, 1e-38)])
def test_scores_of_every_size(dev, shape, dtype, size):
    # queries whose scores leave one token a row, or all of them alike
    bt = batch(shape, dtype, 58)
    assert_plan(bt, shape)
    bt.q = (bt.q.float().clamp(-1.5, 1.5) * size).to(dtype)
    check_attention(dev, bt)


@pytest.mark.parametrize("shape", ["16", "16-joined", "128-64", "128-128-joined", "256-128"])
@pytest.mark.parametrize("power", [-100, -64, 64, 100])
def test_key_scales_of_every_size(dev, shape, power):
    # queries and key scales far from one on opposite sides: the same scores, and the same choice
    # between pages, at every tile height; and a page of keys that are all zero
    bt = batch(shape, BF, 59)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    bt.q = (bt.q.float() * 2.0 ** power).to(BF)
    for pages in bt.pages:
        for i, p in enumerate(pages):
            bt.cache.ks[p] *= 2.0 ** -power * (1.0, 4.0, 0.25)[i % 3]
        if len(pages) > 4:
            bt.cache.ks[pages[3]] = 0
    check_attention(dev, bt, filled=False)


@pytest.mark.parametrize("shape", ["16", "16-joined", "128-64", "128-128-joined", "256-128"])
def test_non_finite_queries_that_see_nothing(dev, shape):
    # zeros where there is no page to see, as for any other query; NaN where there is one
    from my_int4 import _C
    bt = batch(shape, BF, 60)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    bt.q[::3, :, 0] = math.nan
    bt.q[1::3, :, -1] = math.inf
    table, lens, cu = bt.meta(dev)
    table[0] = -1
    out = _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, lens, cu_q=cu).float().cpu()
    assert not out[:bt.n[0]].any()
    bad = torch.arange(sum(bt.n)) % 3 < 2
    seen = torch.arange(sum(bt.n)) >= bt.n[0]
    assert torch.equal(torch.isnan(out).all(-1).all(-1), bad & seen) and torch.equal(torch.isnan(out).any(-1).any(-1), bad & seen)


@pytest.mark.parametrize("shape", ["16", "16-joined", "128-64", "128-128-joined", "256-128"])
@pytest.mark.parametrize("cap", [256.0, 257.0, 1e3, 1e5, 1e7, 1e30, 3e38])
@pytest.mark.parametrize("size", [1.0, 40.0])
def test_wide_caps(dev, shape, cap, size):
    """Caps far above the scores leave them as they are.  A capped score may be off by
    2^-22 of a cap up to 256, else by 2^-20 of itself: twice what the bound without a cap has for the
    rounding of scores and exponents, on scores that a cap only makes smaller."""
    bt = batch(shape, HF, 61, size=1.0)
    assert_plan(bt, shape)
    bt.fill(bt.lens)
    bt.q = (bt.q.float() * size).to(HF)
    out, q, at = run(dev, bt, cap=cap), bt.q.to(dev), 0
    for b, n in enumerate(bt.n):
        ref, A, _ = reference(dev, bt, b, q[at:at + n], cap=cap)
        E = 2 * reference(dev, bt, b, q[at:at + n])[2] + (2.0 ** -22 * cap if cap <= 256 else 0.0)
        assert bool((E < 1 / 16).all())
        assert within(out[at:at + n].double(), ref, plain.attention_bound(ref, A, E, HF)), b
        at += n
