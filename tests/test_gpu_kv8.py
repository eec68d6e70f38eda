"""The 8-bit paged cache on the GPU: what append writes equals the plain form
bit for bit; attention lies within its derived bound of the fp64 value."""
from __future__ import annotations

import math

import pytest
import torch

import _int8 as plain

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def starts(n):
    cu = [0]
    for v in n:
        cu.append(cu[-1] + v)
    return cu


class Batch:
    """Sequences with pages in a random order, garbage and NaN scales in every page
    that is not theirs, -1 behind the tables' ends."""

    def __init__(self, seed, lens, n, Hq, Hkv, D, page, dtype, spare=3, room=0, rot=None, size=1.0):
        g = self.g = gen(seed)
        self.lens, self.n, self.Hq, self.Hkv, self.D, self.page, self.dtype = lens, n, Hq, Hkv, D, page, dtype
        per = [-(-m // page) for m in lens]
        ids = torch.randperm(sum(per) + spare, generator=g).tolist()
        self.pages, at = [], 0
        for m in per:
            self.pages.append(ids[at:at + m])
            at += m
        self.cache = plain.Cache(sum(per) + spare, Hkv, page, D, fill=77)
        width = max(max(per) + room, 1)
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, p in enumerate(self.pages):
            self.table[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        self.cos_sin = plain.table_of(max(max(lens), 1), D if rot is None else rot)
        T = sum(n)
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * size
        qkv[:, Hq:Hq + Hkv] *= torch.exp(0.5 * torch.randn(Hkv, D, generator=g))
        self.qkv = qkv.to(dtype)
        self.q, self.k, self.v = self.qkv.split([Hq, Hkv, Hkv], 1)

    def fill(self, upto):
        """Tokens [0, upto[b]) of each sequence, put there in two steps."""
        for b, m in enumerate(upto):
            for lo, hi in ((0, m // 2), (m // 2, m)):
                x = torch.randn(2, hi - lo, self.Hkv, self.D, generator=self.g) * torch.exp(0.3 * torch.randn(1, generator=self.g))
                self.cache.append(self.pages[b], lo, x[0], x[1])

    def meta(self, dev, ragged=True):
        return self.table.to(dev), i32(self.lens, dev), i32(starts(self.n), dev) if ragged else None


# ------------------------------------------------------------------- append
def check_append(dev, bt, interleaved, ragged, times=1, move=lambda t: t):
    from my_int4 import _C
    start = [m - k for m, k in zip(bt.lens, bt.n)]
    bt.fill([max(s, 0) for s in start])
    gpu = bt.cache.to(dev)
    table, lens, cu = bt.meta(dev, ragged)
    q, k, v = (move(t.to(dev)) for t in (bt.q, bt.k, bt.v))
    for _ in range(times):
        out = _C.kv8_append(q, k, v, bt.cos_sin.to(dev), *gpu, table, lens, cu_q=cu, interleaved=interleaved)
    at = 0
    for b, (s, m) in enumerate(zip(start, bt.n)):
        pos = s + torch.arange(m)
        kk = plain.rotate(bt.k[at:at + m], pos, bt.cos_sin, interleaved)
        ok = pos >= 0
        bt.cache.append(bt.pages[b], max(s, 0), kk[ok], bt.v[at:at + m].float()[ok])
        expect = plain.rotate(bt.q[at:at + m], pos, bt.cos_sin, interleaved).to(bt.dtype)
        assert torch.equal(out[at:at + m].cpu().view(torch.int16), expect.view(torch.int16)), b
        at += m
    for name, a, e in zip(("k", "v", "ks", "vs"), gpu, bt.cache.tensors()):
        a = a.cpu()
        assert torch.equal(torch.nan_to_num(a.float(), nan=-9.0), torch.nan_to_num(e.float(), nan=-9.0)), \
            (name, (a != e).nonzero()[:4])
    return gpu


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,page,rot,interleaved", [(128, 16, 128, False), (64, 64, 64, False), (128, 128, 64, True),
                                                    (64, 32, 16, False), (128, 64, 0, False), (64, 128, 64, True),
                                                    (128, 32, 16, True)])
def test_append_ragged(dev, dtype, D, page, rot, interleaved):
    # prompts and single tokens, pages begun, continued and ended, a sequence with nothing new
    lens, n = [page, 2 * page + 1, 1, 5 * page + 3, page // 2 + 9, 40, 3 * page], [page, 2, 1, 3 * page, 9, 0, 1]
    check_append(dev, Batch(D + page + rot, lens, n, 4, 2, D, page, dtype, rot=rot), interleaved, True, times=2)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 8, 64), (16, 1, 128), (7, 1, 64), (10, 5, 128)])
def test_append_one_token_each(dev, page, Hq, Hkv, D):
    lens = [1, 2, page, page + 1, page - 1, 3 * page // 2, 1000]
    check_append(dev, Batch(page + D, lens, [1] * 7, Hq, Hkv, D, page, BF), False, False, times=3)


@pytest.mark.parametrize("page", [16, 64])
def test_scale_grows_step_by_step(dev, page):
    # token after token with growing values: every step rescales the page
    from my_int4 import _C
    bt = Batch(5, [page], [page], 2, 2, 64, page, BF, rot=0)
    grow = (torch.arange(1, page + 1).float() / 4).view(-1, 1, 1)
    bt.k, bt.v = (bt.k * grow).to(BF), (bt.v / grow).to(BF)
    gpu = bt.cache.to(dev)
    cs = torch.zeros(1, 0, device=dev)
    for i in range(page):
        _C.kv8_append(bt.q[i:i + 1].to(dev), bt.k[i:i + 1].to(dev), bt.v[i:i + 1].to(dev), cs, *gpu, bt.table.to(dev), i32([i + 1], dev))
        bt.cache.append(bt.pages[0], i, bt.k[i:i + 1].float(), bt.v[i:i + 1].float())
    for a, e in zip(gpu, bt.cache.tensors()):
        p = bt.pages[0]
        assert torch.equal(a.cpu()[p], e[p])


def test_append_strides(dev):
    # q, k, v as views of one tensor, and as copies that the kernel cannot read in place
    for move in (lambda t: t, lambda t: t.contiguous(), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.nn.functional.pad(t, (3, 5))[..., 3:-5], lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        check_append(dev, Batch(9, [20, 33], [20, 3], 4, 2, 64, 16, HF), False, True, move=move)


def test_append_special_values(dev):
    bt = Batch(11, [40, 40, 40, 24], [40, 8, 40, 24], 2, 2, 64, 16, BF, rot=0)
    bt.k[3, 0, 7] = math.inf
    bt.v[20, 1, 0] = math.nan
    bt.k[48 + 16:48 + 32] = 0                       # a page of zeros
    bt.v[48 + 16:48 + 32] = 2.0 ** -60              # below the smallest scale
    bt.v[48:48 + 16] = torch.finfo(BF).max
    check_append(dev, bt, False, True, times=2)


def test_append_to_no_page(dev):
    # page numbers out of range and positions behind the table: nothing is written there
    bt = Batch(12, [40, 50, 20], [40, 20, 20], 2, 1, 64, 16, BF)
    bt.pages[0][1] = bt.table[0, 1] = 10 ** 6
    bt.pages[1][3] = bt.table[1, 3] = -7
    bt.table = bt.table[:, :3].contiguous()
    bt.pages = [p[:3] for p in bt.pages]
    check_append(dev, bt, False, True)


def test_append_more_new_tokens_than_length(dev):
    # a length shorter than the new tokens: those before position 0 are left out
    bt = Batch(13, [20, 5], [24, 5], 2, 2, 64, 16, BF)
    check_append(dev, bt, False, True)


def test_append_many_sequences(dev):
    g = gen(3)
    n = torch.randint(0, 40, (150,), generator=g).tolist()
    lens = [k + int(torch.randint(0, 70, (1,), generator=g)) for k in n]
    check_append(dev, Batch(14, lens, n, 2, 1, 64, 16, HF), False, True)


def test_begun_page_forgets_its_past(dev):
    # a page used before, with a NaN scale, begun anew
    bt = Batch(15, [16], [16], 2, 2, 64, 16, BF)
    assert torch.isnan(bt.cache.ks).all()
    gpu = check_append(dev, bt, False, True)
    assert torch.isfinite(gpu[2].cpu()[bt.pages[0]]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (128, 128), (64, 32)])
def test_read(dev, dtype, D, page):
    from my_int4 import _C
    c = plain.Cache(6, 3, page, D)
    g = gen(D)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, generator=g))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, generator=g))
    c.ks.copy_(torch.rand(6, 3, generator=g))
    c.vs.copy_(torch.rand(6, 3, generator=g))
    ids = [4, 0, 4, 5, -1, 6]
    k, v = (t.cpu() for t in _C.kv8_read(*c.to(dev), i32(ids, dev), dtype))
    assert k.shape == v.shape == (6, 3, page, D) and k.dtype == v.dtype == dtype
    assert torch.equal(k[:4], (c.k[ids[:4]].float() * c.ks[ids[:4]][..., None, None]).to(dtype))
    assert torch.equal(v[:4], (c.v[ids[:4]].float() * c.vs[ids[:4]][..., None, None]).to(dtype).transpose(2, 3))
    assert torch.isnan(k[4:].float()).all() and torch.isnan(v[4:].float()).all()
    assert _C.kv8_read(*c.to(dev), i32([], dev), dtype)[0].shape == (0, 3, page, D)


# ---------------------------------------------------------------- attention
def check_attention(dev, bt, window=0, cap=0.0, ragged=True, max_len=0, scale=None, filled=True, move=lambda t: t):
    from my_int4 import _C
    if filled:
        bt.fill(bt.lens)
    q = bt.q
    table, lens, cu = bt.meta(dev, ragged)
    kw = {} if scale is None else {"scale": scale}
    out = _C.kv8_attention(move(q.to(dev)), *bt.cache.to(dev), table, lens, cu_q=cu, window=window, softcap=cap, max_len=max_len, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    out, at = out.cpu().double(), 0
    room = bt.table.shape[1] * bt.page
    for b, (m, L) in enumerate(zip(bt.n, bt.lens)):
        k, v, seen = bt.cache.sequence(bt.pages[b], min(L, room))
        ref, A, E = plain.attention(q[at:at + m], k, v, seen, L - m, bt.D ** -0.5 if scale is None else scale, window, cap)
        got = out[at:at + m]
        bound = plain.attention_bound(ref, A, E, bt.dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), b
        d = torch.nan_to_num((got - ref).abs())
        assert bool((d <= torch.nan_to_num(bound)).all()), (b, float((d / bound).nan_to_num().max()))
        at += m
    return out


# (query heads, key/value heads, D, page)
LAYOUTS = [(8, 8, 64, 16), (32, 8, 128, 16), (16, 2, 128, 64), (28, 4, 64, 32), (16, 1, 128, 128), (5, 1, 64, 64),
           (48, 2, 64, 16)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv,D,page", LAYOUTS)
def test_one_token_each(dev, dtype, Hq, Hkv, D, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700]
    bt = Batch(Hq + D, lens, [1] * len(lens), Hq, Hkv, D, page, dtype)
    check_attention(dev, bt, ragged=False)
    check_attention(dev, bt, ragged=False, max_len=700, filled=False)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv,D,page", LAYOUTS)
def test_chunks(dev, dtype, Hq, Hkv, D, page):
    lens, n = [1, 5, 64, 200, 130, 33, 300], [1, 5, 64, 7, 130, 0, 129]
    check_attention(dev, Batch(Hq + D + 1, lens, n, Hq, Hkv, D, page, dtype), max_len=300)


@pytest.mark.parametrize("D,page,dtype,cap,window", [(128, 16, BF, 0.0, 0), (64, 64, HF, 0.0, 200), (128, 128, HF, 20.0, 0),
                                                     (64, 32, BF, 0.0, 0)])
def test_chunks_that_fill_the_chip(dev, D, page, dtype, cap, window):
    # many heads: tiles of 256 rows, whose wavefronts work in two shifted halves;
    # lengths on both sides of a tile and of the 64 pages that a lane's half holds
    lens, n = [300, 64, 1, 65, 2100, 129], [300, 64, 1, 65, 70, 128]
    check_attention(dev, Batch(D + page, lens, n, 64, 32, D, page, dtype), cap=cap, window=window, max_len=2100)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_chunk_behind_a_long_context_is_split(dev, dtype):
    # few new tokens behind many: 128-row tiles, stretches of the cache joined
    for window in (0, 1500):
        bt = Batch(31, [6000, 150, 4097], [70, 150, 65], 8, 2, 64, 16, dtype)
        out = check_attention(dev, bt, window=window, max_len=6000)
        assert torch.equal(out, check_attention(dev, bt, window=window, max_len=6000, filled=False))


def test_negative_scale(dev):
    for n, ragged in (([1, 1], False), ([60, 70], True)):
        check_attention(dev, Batch(32, [60, 70], n, 8, 2, 64, 16, HF), scale=-0.2, ragged=ragged)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 129, 5000])
@pytest.mark.parametrize("ragged", [False, True])
def test_window(dev, window, ragged):
    lens = [1, 64, 130, 600, 999, 257]
    n = [1, 64, 100, 300, 1, 2] if ragged else [1] * 6
    check_attention(dev, Batch(window, lens, n, 8, 2, 64, 16, HF), window=window, ragged=ragged)


@pytest.mark.parametrize("cap", [5.0, 30.0])
@pytest.mark.parametrize("ragged", [False, True])
def test_softcap(dev, cap, ragged):
    lens, n = [300, 70], [200, 70] if ragged else [1, 1]
    for dtype, D, window in ((BF, 128, 0), (HF, 64, 50)):
        bt = Batch(3, lens, n, 8, 2, D, 32, dtype, size=4.0)
        check_attention(dev, bt, cap=cap, window=window, ragged=ragged)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 1, 128, 64), (4, 4, 64, 16)])
def test_long_cache_is_split(dev, Hq, Hkv, D, page):
    bt = Batch(4, [20001, 3], [1, 1], Hq, Hkv, D, page, BF)
    out = check_attention(dev, bt, ragged=False)
    again = check_attention(dev, bt, ragged=False, filled=False)
    assert torch.equal(out, again)


@pytest.mark.parametrize("B", [33, 128, 129])
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (40, 2), (9, 9)])
def test_many_sequences_over_a_long_cache(dev, B, Hq, Hkv):
    # taken by length, up to 128 of them: equal lengths, empty sequences, a round of
    # the CUs that ends inside the batch, two workgroups a head (20 query rows)
    lens = [(1100, 0, 70, 1, 64, 70, 300, 129)[b % 8 if b % 40 else 0] if b % 8 or b % 40 == 0 else 65 for b in range(B)]
    bt = Batch(B + Hq, lens, [1] * B, Hq, Hkv, 64, 64, BF)
    check_attention(dev, bt, ragged=False, max_len=1100)
    check_attention(dev, bt, ragged=False, window=1030, filled=False)


def test_bound_of_lengths_only_splits(dev):
    # a bound below the true lengths costs speed, not tokens; a window over a long cache
    bt = Batch(6, [5000, 300], [1, 1], 8, 2, 64, 16, BF)
    check_attention(dev, bt, ragged=False, max_len=64)
    check_attention(dev, bt, ragged=False, max_len=5000, filled=False)
    check_attention(dev, bt, ragged=False, window=700, filled=False)


def test_rows_that_see_nothing(dev):
    # length 0; more queries than tokens (positions before 0); no page at all
    from my_int4 import _C
    bt = Batch(7, [0, 3, 40], [2, 6, 40], 4, 2, 64, 16, BF)
    out = check_attention(dev, bt)
    assert torch.equal(out[:2], torch.zeros_like(out[:2])) and torch.equal(out[2:5], torch.zeros_like(out[2:5]))
    assert out[5].abs().sum() > 0
    table = torch.full_like(bt.table, -1).to(dev)
    out = _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, i32(bt.lens, dev), cu_q=i32(starts(bt.n), dev))
    assert torch.equal(out, torch.zeros_like(out))
    none = _C.kv8_attention(bt.q[:3].to(dev), *bt.cache.to(dev), table[:, :0].contiguous(), i32(bt.lens, dev))
    assert torch.equal(none, torch.zeros_like(none))


def test_missing_pages_are_not_seen(dev):
    for ragged, n in ((True, [90, 130]), (False, [1, 1])):
        bt = Batch(8, [100, 130], n, 8, 2, 128, 16, HF)
        bt.fill(bt.lens)
        bt.pages[0][2] = bt.table[0, 2] = -1
        bt.pages[0][0] = bt.table[0, 0] = 2 ** 30
        bt.pages[1][8] = bt.table[1, 8] = bt.cache.k.shape[0]
        check_attention(dev, bt, ragged=ragged, filled=False)


def test_length_behind_the_table(dev):
    for ragged, n in ((True, [30, 5]), (False, [1, 1])):
        bt = Batch(81, [64, 64], n, 4, 1, 64, 16, HF)
        bt.fill(bt.lens)
        bt.table = bt.table[:, :3].contiguous()
        bt.pages = [p[:3] for p in bt.pages]
        check_attention(dev, bt, ragged=ragged, filled=False)


@pytest.mark.parametrize("dtype,values", [(BF, (1e30, 1e-30, 3e38, 1e-38, 0.0)), (HF, (6e4, 1e-5, 6e-8, 1.0, 0.0))])
def test_extreme_queries(dev, dtype, values):
    # scores of every size; the scale takes them back where they would all saturate
    for v in values:
        bt = Batch(10, [70, 40], [1, 1], 4, 2, 64, 16, dtype)
        bt.q = (bt.q.float().clamp(-1, 1) * v).to(dtype)
        check_attention(dev, bt, ragged=False, scale=0.125 / v if 0 < v < 1e30 and v > 1e-30 else None)


def test_non_finite_values(dev):
    # a query, and a page's scale, that are not finite: NaN for the rows that see them only
    bt = Batch(16, [100, 100], [100, 100], 4, 2, 64, 16, BF)
    bt.fill(bt.lens)
    bt.q[150, 1, 3] = math.nan
    bt.q[151, 2, 9] = math.inf
    bt.cache.vs[bt.pages[0][3], 1] = math.nan
    from my_int4 import _C
    table, lens, cu = bt.meta(dev)
    out = _C.kv8_attention(bt.q.to(dev), *bt.cache.to(dev), table, lens, cu_q=cu).cpu()
    expect = torch.zeros(200, 4, dtype=torch.bool)
    expect[48:100, 2:] = True                       # heads 2, 3 use key/value head 1, from its page's first token on
    expect[150, 1] = expect[151, 2] = True
    assert torch.equal(torch.isnan(out.float()).all(-1), expect) and torch.equal(torch.isnan(out.float()).any(-1), expect)
    one = _C.kv8_attention(bt.q[[99, 199]].to(dev), *bt.cache.to(dev), table, lens).cpu()
    assert torch.isnan(one[0, 2:].float()).all() and torch.isfinite(one[0, :2].float()).all() and torch.isfinite(one[1].float()).all()


def test_scales_of_every_size(dev):
    # pages of zeros, of tiny and of large values side by side
    for ragged, n in ((True, [64, 30]), (False, [1, 1])):
        bt = Batch(17, [64, 150], n, 4, 2, 64, 16, BF)
        bt.fill(bt.lens)
        p = bt.pages[1]
        for i, f in ((0, 0.0), (1, 2.0 ** -20), (2, 2.0 ** 20), (3, 2.0 ** -39)):
            if f:
                bt.cache.vs[p[i]] *= f
            else:
                bt.cache.v[p[i]] = 0
                bt.cache.vs[p[i]] = plain.FLOOR
            bt.cache.ks[p[i]] *= 0.5
        bt.cache.ks[bt.pages[0][1]] *= 40             # scores in the hundreds
        check_attention(dev, bt, ragged=ragged, filled=False)


def test_query_strides(dev):
    for move in (lambda t: t, lambda t: torch.nn.functional.pad(t, (8, 8))[..., 8:-8], lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2],
                 lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        check_attention(dev, Batch(18, [50, 20], [50, 3], 4, 2, 64, 16, BF), move=move)


def test_offsets_past_32_bits(dev):
    # the last pages of a cache of more than 2^31 codes a tensor
    from my_int4 import _C
    Hkv, D, page = 8, 128, 128
    pages = (2 ** 31 // (Hkv * D * page)) + 300
    small = Batch(19, [300], [300], 8, Hkv, D, page, BF, spare=0)
    small.fill([250])
    k = torch.zeros(pages, Hkv, page, D, dtype=torch.int8, device=dev)
    v = torch.zeros(pages, Hkv, D, page, dtype=torch.int8, device=dev)
    ks, vs = (torch.full((pages, Hkv), math.nan, device=dev) for _ in range(2))
    at = [pages - 1, 1, pages - 2]
    for t, c in zip((k, v, ks, vs), small.cache.tensors()):
        t[at] = c[small.pages[0]].to(dev)
    table = i32([at], dev)
    q, kn, vn = (t[250:].to(dev) for t in (small.q, small.k, small.v))
    cu, lens = i32([0, 50], dev), i32([300], dev)
    qr = _C.kv8_append(q, kn, vn, small.cos_sin.to(dev), k, v, ks, vs, table, lens, cu_q=cu)
    pos = torch.arange(250, 300)
    small.cache.append(small.pages[0], 250, plain.rotate(small.k[250:], pos, small.cos_sin, False), small.v[250:].float())
    for t, c in zip((k, v, ks, vs), small.cache.tensors()):
        assert torch.equal(t[at].cpu(), c[small.pages[0]])
    kr, vr = _C.kv8_read(k, v, ks, vs, i32(at, dev), BF)
    assert torch.equal(vr[2].cpu(), (small.cache.v[small.pages[0][2]].float() * small.cache.vs[small.pages[0][2]][:, None, None]).to(BF).transpose(1, 2))
    kk, vv, seen = small.cache.sequence(small.pages[0], 300)
    for rows, c in ((qr, cu), (qr[-1:], None)):
        ref, A, E = plain.attention(rows.cpu(), kk, vv, seen, 300 - rows.shape[0], D ** -0.5)
        out = _C.kv8_attention(rows, k, v, ks, vs, table, lens, cu_q=c).cpu().double()
        assert bool(((out - ref).abs() <= plain.attention_bound(ref, A, E, BF)).all())


def test_graph_replays_follow_the_lengths(dev):
    # a captured decode step: append and attention, lengths advanced between replays
    from my_int4 import _C
    Hq, Hkv, D, page, steps = 8, 2, 64, 16, 6
    lens0 = [5, 14, 31, 200]
    bt = Batch(20, [m + steps for m in lens0], [steps] * 4, Hq, Hkv, D, page, BF)
    bt.fill(lens0)
    gpu, cs, table = bt.cache.to(dev), bt.cos_sin.to(dev), bt.table.to(dev)
    new = [t.view(4, steps, -1, D) for t in (bt.q, bt.k, bt.v)]
    q, k, v = (t[:, 0].contiguous().to(dev) for t in new)
    lens = i32([m + 1 for m in lens0], dev)
    kept = [t.clone() for t in gpu]

    def step():
        qr = _C.kv8_append(q, k, v, cs, *gpu, table, lens)
        return qr, _C.kv8_attention(qr, *gpu, table, lens)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = step()
    for t, c in zip(gpu, kept):
        t.copy_(c)
    for i in range(steps):
        for dst, src in zip((q, k, v), new):
            dst.copy_(src[:, i])
        lens.fill_(0)
        lens.add_(i32([m + i + 1 for m in lens0], dev))
        graph.replay()
        torch.cuda.synchronize()
        for b, m in enumerate(lens0):
            pos = torch.tensor([m + i])
            bt.cache.append(bt.pages[b], m + i, plain.rotate(new[1][b, i:i + 1], pos, bt.cos_sin, False), new[2][b, i:i + 1].float())
            kk, vv, seen = bt.cache.sequence(bt.pages[b], m + i + 1)
            ref, A, E = plain.attention(qr[b:b + 1].cpu(), kk, vv, seen, m + i, D ** -0.5)
            assert bool(((out[b:b + 1].cpu().double() - ref).abs() <= plain.attention_bound(ref, A, E, BF)).all()), (i, b)
        eager = _C.kv8_attention(qr, *gpu, table, lens)
        assert torch.equal(eager, out)


def test_side_stream(dev):
    from my_int4 import _C
    bt = Batch(21, [3000, 70], [1, 1], 8, 2, 64, 16, BF)
    bt.fill(bt.lens)
    table, lens, _ = bt.meta(dev)
    args = (bt.q.to(dev), *bt.cache.to(dev), table, lens)
    expect = _C.kv8_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_C.kv8_attention(*args) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(o, expect) for o in outs)


def test_refusals(dev):
    from my_int4 import _C
    bt = Batch(22, [20, 20], [1, 1], 4, 2, 64, 16, BF)
    cache, (table, lens, _) = bt.cache.to(dev), bt.meta(dev)
    q, k, v, cs = bt.q.to(dev), bt.k.to(dev), bt.v.to(dev), bt.cos_sin.to(dev)
    kc, vc, ks, vs = cache

    def append(q=q, k=k, v=v, cs=cs, cache=cache, table=table, lens=lens, **kw):
        return _C.kv8_append(q, k, v, cs, *cache, table, lens, **kw)

    def attend(q=q, cache=cache, table=table, lens=lens, **kw):
        return _C.kv8_attention(q, *cache, table, lens, **kw)

    wide = torch.zeros(4, 2, 16, 96, dtype=torch.int8, device=dev)
    odd = torch.zeros(4, 2, 24, 64, dtype=torch.int8, device=dev)
    bad = [
        ("bf16 or fp16", lambda: append(q=q.float())), ("one type", lambda: append(k=k.half())),
        ("tokens, heads, head_dim", lambda: append(q=q[0])), ("must agree", lambda: append(k=k[:, :1], v=v[:, :1])),
        ("must agree", lambda: append(k=k[:1], v=v[:1])), ("multiple of 16", lambda: append(cs=cs[:, :24].contiguous())),
        ("fp32", lambda: append(cs=cs.double())), ("int32", lambda: append(table=table.long())),
        ("int32", lambda: append(lens=lens.long())), ("sequences", lambda: append(lens=lens[:1])),
        ("one new token per sequence", lambda: append(q=q[:1], k=k[:1], v=v[:1])),
        (r"sequences \+ 1", lambda: append(cu_q=i32([0, 1], dev))), ("CUDA", lambda: append(q=q.cpu())),
        ("CUDA", lambda: append(table=table.cpu())), ("k_cache must be contiguous int8", lambda: append(cache=(kc.float(), vc, ks, vs))),
        ("v_cache must be", lambda: append(cache=(kc, kc, ks, vs))), ("k_scale and v_scale", lambda: append(cache=(kc, vc, ks[:1], vs))),
        ("head_dim must be", lambda: _C.kv8_read(wide, wide.transpose(2, 3).contiguous(), ks[:4], vs[:4], i32([0], dev))),
        ("page_size must be", lambda: _C.kv8_read(odd, odd.transpose(2, 3).contiguous(), ks[:4], vs[:4], i32([0], dev))),
        ("multiple of the cache", lambda: attend(q=q[:, :3])), ("head_dim", lambda: attend(q=q[..., :32])),
        ("negative", lambda: attend(window=-1)), ("negative", lambda: attend(max_len=-1)), ("softcap", lambda: attend(softcap=-1.0)), ("scale must be finite", lambda: attend(scale=math.inf)),
        ("softcap", lambda: attend(softcap=math.inf)), ("bf16 or fp16", lambda: attend(q=q.float())),
        ("one new token per sequence", lambda: attend(q=torch.cat((q, q)))),
        ("bf16 or fp16", lambda: _C.kv8_read(*cache, i32([0], dev), torch.float32)),
        ("int32", lambda: _C.kv8_read(*cache, torch.zeros(1, dtype=torch.int64, device=dev))),
    ]
    for text, call in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
