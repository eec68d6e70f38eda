"""The 8-bit paged cache at the ends of its arguments' ranges."""
from __future__ import annotations

import pytest
import torch

import _int8 as plain
from test_gpu_kv8 import BF, HF, Batch, check_attention, i32

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


# (query heads, key/value heads, new tokens of the sequences): 16-, 128- and 256-row tiles
@pytest.mark.parametrize("rows,Hq,Hkv,D,n", [(16, 8, 2, 64, [3, 0, 20]), (128, 64, 4, 64, [150, 65, 200]), (256, 64, 1, 128, [420, 690, 500])])
@pytest.mark.parametrize("before,behind", [(0, 1), (0, 40), (5, 0), (37, 130)])
def test_tokens_of_no_sequence_are_zeros(dev, rows, Hq, Hkv, D, n, before, behind):
    # a batch with room for more tokens than its sequences have, before their first and behind their last
    from my_int4 import _C
    from wush_int4_kernel_amd import capi
    lens = [k + 70 for k in n]
    bt = Batch(43, lens, n, Hq, Hkv, D, 64, BF)
    bt.fill([70] * 3)
    T = before + sum(n) + behind
    assert capi.kv8_attention_plan(bt.cache.k.shape[0], Hkv, 64, D, 3, T, True, Hq, bt.table.shape[1])[0] == rows
    table, lens, cu = bt.meta(dev)
    gpu, cs = bt.cache.to(dev), bt.cos_sin.to(dev)
    whole = torch.full((T, Hq + 2 * Hkv, D), float("nan"), dtype=BF)
    whole[before:T - behind] = bt.qkv
    outs = []
    for t, c in ((bt.qkv, cu), (whole, cu + before)):
        q, k, v = t.to(dev).split([Hq, Hkv, Hkv], 1)
        dirty = [torch.full((T * Hq * D,), float("nan"), dtype=BF, device=dev) for _ in range(4)]
        del dirty                                     # what the outputs' memory may hold
        qr = _C.kv8_append(q, k, v, cs, *gpu, table, lens, cu_q=c)
        outs.append((qr, _C.kv8_attention(qr, *gpu, table, lens, cu_q=c, max_len=max(bt.lens)), [t.clone() for t in gpu]))
    for a, b in zip(outs[0][2], outs[1][2]):          # the same cache
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))
    for a, b in zip(*(o[:2] for o in outs)):
        assert torch.equal(a, b[before:T - behind])
        assert not b[:before].any() and not b[T - behind:].any()


def test_no_sequence_at_all(dev):
    from my_int4 import _C
    bt = Batch(44, [20], [20], 4, 2, 64, 16, BF)
    gpu, cs = bt.cache.to(dev), bt.cos_sin.to(dev)
    q, k, v = (t.to(dev) for t in (bt.q, bt.k, bt.v))
    kept = [t.clone() for t in gpu]
    for table, lens, cu in ((bt.table[:0], [], [0]), (bt.table, [20], [0, 0]), (bt.table, [20], [20, 20])):
        args = table.to(dev), i32(lens, dev)
        assert not _C.kv8_append(q, k, v, cs, *gpu, *args, cu_q=i32(cu, dev)).any()
        assert not _C.kv8_attention(q, *gpu, *args, cu_q=i32(cu, dev)).any()
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(gpu, kept))


# (rows of a tile, head_dim, query heads, key/value heads, new tokens, sequences' lengths)
@pytest.mark.parametrize("rows,D,Hq,Hkv,n", [(16, 128, 8, 2, [1, 1]), (16, 64, 16, 1, [1, 1]), (16, 128, 8, 2, [5, 9]), (128, 64, 64, 4, [300, 130])])
@pytest.mark.parametrize("times,keys", [(20, 1.0), (100, 1.0), (300, 1.0), (1000, 0.0), (4000, 0.0)])
def test_queries_with_an_outlier_channel(dev, rows, D, Hq, Hkv, n, times, keys):
    """One channel of q many times the others, with keys as elsewhere or none: the other
    channels' part of the scores stays.  q may be off by 2^-23 of its row's largest value."""
    from my_int4 import _C
    from wush_int4_kernel_amd import capi
    lens = [700, 500]
    bt = Batch(45, lens, n, Hq, Hkv, D, 64, HF)
    bt.fill(lens)
    bt.cache.k[..., 5] = (bt.cache.k[..., 5] * keys).to(torch.int8)
    bt.q = bt.q.clone()
    bt.q[..., 5] = times * torch.sign(bt.q[..., 5])
    ragged = n != [1, 1]
    assert capi.kv8_attention_plan(bt.cache.k.shape[0], Hkv, 64, D, 2, sum(n), ragged, Hq, bt.table.shape[1])[0] == rows
    table, lens, cu = bt.meta(dev, ragged)
    out = _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, lens, cu_q=cu).cpu().double()
    at = 0
    for b, m in enumerate(n):
        q = bt.q[at:at + m]
        k, v, seen = bt.cache.sequence(bt.pages[b], bt.lens[b])
        ref, A, E = plain.attention(q, k, v, seen, bt.lens[b] - m, D ** -0.5)
        most = k.abs().sum(-1).amax(0).repeat_interleave(Hq // Hkv)                        # (Hq,): of a token's keys, summed
        E = E + (2.0 ** -23 * q.double().abs().amax(-1) * most * D ** -0.5)[..., None]
        assert bool(((out[at:at + m] - ref).abs() <= plain.attention_bound(ref, A, E, HF)).all()), b
        at += m


def test_reading_more_pages_than_a_launch(dev):
    # 2^22 (page, head)s are one launch, and 2^23 have 2^32 threads; 34 GB of output
    from my_int4 import _C
    H, n = 2 ** 9, 2 ** 14 + 5
    g = torch.Generator().manual_seed(46)
    c = plain.Cache(3, H, 16, 64)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, generator=g))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, generator=g))
    c.ks.copy_(torch.rand(3, H, generator=g))
    c.vs.copy_(torch.rand(3, H, generator=g))
    ids = (torch.arange(n) * 7 % 3).to(torch.int32)
    k, v = _C.kv8_read(*c.to(dev), ids.to(dev), BF)
    kr = (c.k.float() * c.ks[..., None, None]).to(BF).to(dev)
    vr = (c.v.float() * c.vs[..., None, None]).to(BF).transpose(2, 3).contiguous().to(dev)
    for at in (0, 2 ** 13 - 2, 2 ** 14 - 2, n - 5):
        i = ids[at:at + 5].long().to(dev)
        assert torch.equal(k[at:at + 5], kr[i]) and torch.equal(v[at:at + 5], vr[i])
    del k, v
    torch.cuda.empty_cache()
