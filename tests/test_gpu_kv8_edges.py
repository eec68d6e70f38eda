"""The 8-bit paged cache at the ends of its arguments' ranges."""
from __future__ import annotations

import pytest
import torch

import _int8 as plain
from test_gpu_kv8 import BF, Batch, check_attention, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ragged", [False, True])
def test_length_beyond_the_longest(dev, ragged):
    # a table with room for 2^31 tokens: lengths up to 2^30 count, longer ones as none
    from my_int4 import _C
    page, width = 128, 2 ** 24 + 1
    bt = Batch(41, [200, 200, 200], [1, 1, 1], 4, 2, 64, page, BF)
    bt.fill(bt.lens)
    table = torch.full((3, width), -1, dtype=torch.int32, device=dev)
    for b, p in enumerate(bt.pages):
        table[b, :len(p)] = i32(p, dev)
    last = 2 ** 30 // page - 1                        # the page of position 2^30 - 1
    table[2, last] = bt.pages[2][0]
    gpu = bt.cache.to(dev)
    lens = i32([200, 2 ** 31 - 1, 2 ** 30], dev)
    cu = i32([0, 1, 2, 3], dev) if ragged else None
    out = _C.kv8_attention(bt.q.to(dev), *gpu, table, lens, cu_q=cu).cpu().double()
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    # of the third, three pages of tokens are seen: its own two, and the last, which is the first again
    for b, (pages, n) in ((0, (bt.pages[0], 200)), (2, (bt.pages[2] + bt.pages[2][:1], 3 * page))):
        k, v, seen = bt.cache.sequence(pages, n)
        ref, A, E = plain.attention(bt.q[b:b + 1], k, v, seen, n - 1, 64 ** -0.5)
        assert bool(((out[b:b + 1] - ref).abs() <= plain.attention_bound(ref, A, E, BF)).all()), b
    kept = [t.clone() for t in gpu]
    q, k, v, cs = (t.to(dev) for t in (bt.q, bt.k, bt.v, bt.cos_sin))
    _C.kv8_append(q, k, v, cs, *gpu, table, i32([2 ** 31 - 1, -1, -2 ** 31], dev), cu_q=cu)
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(gpu, kept))


WIDE = [2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 62]


@pytest.mark.parametrize("window", WIDE)
@pytest.mark.parametrize("Hq,Hkv,lens,n", [(4, 2, [0, 3, 40], [2, 6, 40]), (64, 8, [300, 130, 5], [900, 130, 9]), (8, 8, [5000, 3], [1, 1])])
def test_window_wider_than_every_sequence(dev, window, Hq, Hkv, lens, n):
    # also where more tokens are new than the sequence has (positions below 0)
    bt = Batch(42, lens, n, Hq, Hkv, 64, 16, BF)
    out = check_attention(dev, bt, window=window)
    assert torch.equal(out, check_attention(dev, bt, filled=False))
