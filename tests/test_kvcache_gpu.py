"""The paged key/value cache through its public entry points against plain 64-bit forms of the same operators.

Every slot that no sequence owns, and every slot past a sequence's length, holds NaN (a 4-bit cache: NaN scales):
whatever reaches an output from there shows. Bars, from the arithmetic:

* attention: the kernels round the softmax's probabilities to the 16-bit type before their product with V and the
  result to the output's type; a 4-bit cache's probabilities are FP16. A rounding is off by u |x| on average (u = 2^-9
  in BF16 and 2^-12 in FP16), by 2u |x| at worst; the probabilities' errors average over the keys, and |out| is an
  average of |v| that stays below its maximum. Scores and sums are FP32: with |score| < 64, 2^-24 a step over at most
  128 products and the exponential's 2 ulp stay below 1e-4. So the bar is |error| <= (2u + 1e-4) max |v|.
* rotation: FP32, off by d <= 2^-23 (|x| + |y|), then the nearest value of the 16-bit type: its own distance + 2d.
* 4 bits: a value is within half a step of its code's, and the rounded scale (15 steps of 2^-12 each, relative) and
  minimum (2^-12 |min|) move the range's ends: scale / 2 + 2^-11 (max - min) + 2^-11 |min| + 2^-11 |value|.
"""

import ctypes
import math

import pytest

from jitcast_b200 import _lib

pytestmark = pytest.mark.gpu

ROUNDING = {"bf16": 2.0 ** -9, "fp16": 2.0 ** -12}


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kvcache(jc):
    from jitcast_b200 import kvcache

    return kvcache


def dtype_of(torch, name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def quantise(torch, x):
    """(codes, scales) of x [.., dim] as the header defines them, in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    scale, low = ((hi - lo) / 15).half(), lo.half()
    s, m = scale.double()[..., None], low.double()[..., None]
    code = torch.where(s > 0, (g - m) / s.clamp(min=1e-30), torch.zeros_like(g)).round().clamp(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([scale, low], -1)


def values(torch, codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).double()
    return (c * scales[..., :1].double() + scales[..., 1:].double()).flatten(-2).half().double()


class World:
    """A cache with sequences of given lengths in shuffled pages, and the 64-bit keys and values that it holds."""

    def __init__(self, torch, kvcache, bits, dtype, dim, kv_heads, page, lengths, news, seed=0, spare=3, share=1.0):
        g = torch.Generator().manual_seed(seed)
        self.torch, self.kvcache = torch, kvcache
        self.dt, self.dim, self.kv, self.page, self.bits = dtype_of(torch, dtype), dim, kv_heads, page, bits
        self.lengths, self.news = lengths, news
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(need) + spare, generator=g).tolist()
        cols = max(max(need), 1)
        self.table = torch.full((len(lengths), cols), -1, dtype=torch.int32)
        shape = (sum(need) + spare, kv_heads, page)
        nan = float("nan")
        if bits == 16:
            pools = [torch.full((*shape, dim), nan, dtype=self.dt) for _ in range(2)]
            scales = [None, None]
        else:
            pools = [torch.randint(0, 256, (*shape, dim // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
            scales = [torch.full((*shape, dim // 32, 2), nan, dtype=torch.float16) for _ in range(2)]
        self.held = []  # per sequence (k, v) [length, kv_heads, dim] in 64 bits
        for s, n in enumerate(lengths):
            ids = [order.pop() for _ in range(need[s])]
            self.table[s, :need[s]] = torch.tensor(ids, dtype=torch.int32)
            pair = []
            for which in range(2):
                x = torch.randn((n, kv_heads, dim), generator=g) * share
                if which == 0:
                    x = x + torch.randn((1, kv_heads, dim), generator=g)
                x = x.to(self.dt)
                at = torch.arange(n)
                page_of = torch.tensor(ids + [0])[at // page] if n else at
                if bits == 16:
                    pools[which][page_of, :, at % page] = x
                    pair.append(x.double())
                else:
                    codes, sc = quantise(torch, x)
                    pools[which][page_of, :, at % page] = codes
                    scales[which][page_of, :, at % page] = sc
                    pair.append(values(torch, codes, sc))
            self.held.append(pair)
        self.pools = [t.cuda() for t in pools]
        self.scales = [None if t is None else t.cuda() for t in scales]
        self.cache = kvcache.PagedCache.over(*self.pools, *self.scales)
        self.bounds = [0]
        for n in news:
            self.bounds.append(self.bounds[-1] + n)
        self.tokens = self.bounds[-1]

    def step(self, start=True, max_length=None, max_new=None):
        t = self.torch
        if not start:
            return self.kvcache.Step(t.tensor(self.lengths, dtype=t.int32).cuda(), self.table.cuda(), max(self.lengths))
        return self.kvcache.Step(t.tensor(self.lengths, dtype=t.int32).cuda(), self.table.cuda(),
                                 max(self.lengths) if max_length is None else max_length,
                                 t.tensor(self.bounds, dtype=t.int32).cuda(),
                                 max(self.news) if max_new is None else max_new)

    def expect(self, q, window, sinks, scale=None):
        """The formula on q [tokens, heads, dim] in 64 bits; hidden keys and values are never touched."""
        t = self.torch
        heads = q.shape[1]
        scale = self.dim ** -0.5 if scale is None else scale
        out = t.zeros(q.shape, dtype=t.float64)
        for s, (n, length) in enumerate(zip(self.news, self.lengths)):
            k, v = self.held[s]
            for i in range(n):
                at = length - n + i
                if at < 0:
                    continue
                j = t.arange(at + 1)
                if window:
                    j = j[(j > at - window) | (j < sinks)]
                kk = k[j].repeat_interleave(heads // self.kv, 1)
                vv = v[j].repeat_interleave(heads // self.kv, 1)
                z = t.einsum("hd,jhd->hj", q[self.bounds[s] + i].double(), kk) * scale
                out[self.bounds[s] + i] = t.einsum("hj,jhd->hd", t.softmax(z, -1), vv)
        return out

    def most(self):
        """max |v| of what is finite."""
        m = [h[1][h[1].isfinite()].abs().max() for h in self.held if h[1].numel()]
        return float(max(m)) if m else 0.0


def bar(w, dtype):
    return (2 * ROUNDING[dtype] + 1e-4) * w.most()


def sync():
    _lib.check(_lib.lib().jc_device_sync(0))


def check(torch, w, dtype, heads, window=0, sinks=0, seed=1, start=True, scale=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((w.tokens, heads, w.dim), generator=g).to(w.dt)
    got = w.cache.attention(w.step(start), q.cuda(), window=window, sinks=sinks, scale=scale)
    sync()
    assert got.dtype == w.dt and got.shape == q.shape
    exp = w.expect(q, window, sinks, scale)
    got = got.cpu().double()
    assert not got.isnan().any()
    err = float((got - exp).abs().max()) if exp.numel() else 0.0
    print(f"max error {err:.2e} of a bar of {bar(w, dtype):.2e}")
    assert err <= bar(w, dtype)
    return got


# (heads, kv heads, page, lengths, new tokens, window, sinks)
ONE = [
    (2, 2, 16, [1], [1], 0, 0),
    (3, 3, 64, [5, 1, 16, 17], [1, 1, 1, 1], 0, 0),
    (8, 1, 48, [127, 128, 129, 700], [1, 1, 1, 1], 100, 3),
    (6, 2, 64, [300, 2, 65], [1, 1, 1], 1, 0),
    (12, 4, 32, [1000, 31, 33, 64], [1, 1, 1, 1], 64, 4),
    (5, 1, 128, [2049, 4097], [1, 1], 0, 0),
    (20, 1, 16, [333], [1], 50, 0),
    (40, 2, 64, [900, 5000], [1, 1], 1000, 70),
]
MANY = [
    (2, 2, 64, [130, 130], [130, 130], 0, 0),
    (4, 2, 16, [1, 40, 200], [1, 3, 190], 0, 0),
    (3, 3, 48, [128, 256, 257], [128, 256, 257], 0, 0),
    (6, 2, 64, [500, 77, 300], [33, 0, 300], 40, 0),
    (8, 1, 32, [700, 129], [140, 129], 128, 5),
    (7, 1, 128, [900], [300], 257, 200),
    (2, 1, 64, [0, 3, 5], [0, 3, 9], 0, 0),      # nothing cached; more new tokens than the length: empty rows
    (4, 4, 64, [600], [600], 1, 1),
    (4, 4, 64, [1500, 40], [9, 17], 300, 130),
    (1, 1, 64, [1030], [1000], 0, 0),
    (24, 8, 16, [90, 400, 18], [2, 100, 18], 90, 16),
]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", ONE, ids=str)
def test_one_token_attention(torch, kvcache, case, bits, dtype, dim):
    heads, kv, page, lengths, news, window, sinks = case
    w = World(torch, kvcache, bits, dtype, dim, kv, page, lengths, news)
    a = check(torch, w, dtype, heads, window, sinks)
    b = check(torch, w, dtype, heads, window, sinks, start=False)  # the form without starts
    assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", MANY, ids=str)
def test_many_token_attention(torch, kvcache, case, bits, dtype, dim):
    heads, kv, page, lengths, news, window, sinks = case
    w = World(torch, kvcache, bits, dtype, dim, kv, page, lengths, news)
    check(torch, w, dtype, heads, window, sinks)


# The library takes few rows of few heads to one kernel and many to another: the same cases with 16 (8) times the heads.
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("i", [0, 1, 2, 3, 4, 5, 7, 9, 10])
def test_many_token_attention_of_many_heads(torch, kvcache, i, bits, dim):
    heads, kv, page, lengths, news, window, sinks = MANY[i]
    f = 8 if kv >= 4 else 16
    dtype = "bf16" if (i + bits + dim // 64) % 2 else "fp16"
    w = World(torch, kvcache, bits, dtype, dim, kv * f, page, lengths, news)
    check(torch, w, dtype, heads * f, window, sinks)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page", [256, 592, 1024])
@pytest.mark.parametrize("new", [1, 40])
def test_large_pages(torch, kvcache, bits, page, new):
    w = World(torch, kvcache, bits, "bf16", 64, 2, page, [1300, 40, 593], [new, new, new])
    check(torch, w, "bf16", 4, window=500, sinks=20)
    check(torch, w, "bf16", 4)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_token_of_many_heads_a_kv_head(torch, kvcache, bits, dim):
    # more query rows of one token than the splits take: the tiles, with and without starts
    w = World(torch, kvcache, bits, "fp16", dim, 2, 64, [300, 1, 77], [1, 1, 1])
    a = check(torch, w, "fp16", 80, window=90, sinks=2)
    assert torch.equal(a, check(torch, w, "fp16", 80, window=90, sinks=2, start=False))


@pytest.mark.parametrize("bits", [16, 4])
def test_many_sequences(torch, kvcache, bits):
    # hundreds of sequences, some without new tokens, some without any: every token finds its own
    lengths = [(7 * s) % 50 for s in range(333)]
    news = [min(n, (3 * s) % 4) for s, n in enumerate(lengths)]
    w = World(torch, kvcache, bits, "bf16", 64, 1, 16, lengths, news)
    check(torch, w, "bf16", 2)
    g = torch.Generator().manual_seed(8)
    x = torch.randn((w.tokens, 1, 64), generator=g).to(w.dt).cuda()
    w.cache.append(w.step(), x, x)
    k, v = w.cache.read(w.step(), w.tokens)
    sync()
    if bits == 16:
        assert torch.equal(k, x) and torch.equal(v, x)
    else:
        codes, sc = quantise(torch, x.cpu())
        assert torch.equal(k.cpu().double(), values(torch, codes, sc)) and torch.equal(k, v)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [1, 2, 5, 70])
def test_long_histories(torch, kvcache, bits, new):
    # key ranges split over many blocks and joined; lengths that end inside a page and a tile
    w = World(torch, kvcache, bits, "fp16", 64, 2, 64, [20011, 9, 6007], [new, min(new, 9), new])
    a = check(torch, w, "fp16", 4)
    b = check(torch, w, "fp16", 4)
    assert torch.equal(a, b)  # the same inputs give the same bits
    check(torch, w, "fp16", 4, window=5000, sinks=100)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [64, 48])
def test_many_rows_over_long_histories(torch, kvcache, bits, dim, page):
    # few tiles of rows, whose keys are split over several CTAs and joined; a short sequence beside the long one, a key
    # that not every row sees with an undefined value, and the same bits twice
    w = World(torch, kvcache, bits, "bf16", dim, 8, page, [4500, 200], [70, 45])
    a = check(torch, w, "bf16", 8)
    assert torch.equal(a, check(torch, w, "bf16", 8))
    check(torch, w, "bf16", 8, window=3300, sinks=100)
    where, row = int(w.table[0, 4490 // page]), 4490 % page
    if bits == 16:
        w.pools[1][where, :, row, 5] = float("inf")
    else:
        w.scales[1][where, :, row, 0] = float("nan")
    g = torch.Generator().manual_seed(1)
    q = torch.randn((w.tokens, 8, dim), generator=g).to(w.dt)
    got = w.cache.attention(w.step(), q.cuda()).cpu().double()
    sync()
    assert float((got[:60] - a[:60]).abs().max()) <= 2 * bar(w, "bf16")  # tokens before it
    assert not bool(got[60:70, :, 5].isfinite().any())
    w.table[0, 20] = -7  # and a page outside the pool: reported, its keys left out
    got = w.cache.attention(w.step(), q.cuda()).cpu().double()
    with pytest.raises(_lib.JcArgumentError):
        sync()
    assert bool(got[:60].isfinite().all())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_peaked_scores(torch, kvcache, bits, new):
    # scores over a wide range: the running maximum moves often and late
    w = World(torch, kvcache, bits, "bf16", 64, 1, 64, [777], [new], share=4.0)
    check(torch, w, "bf16", 2, scale=0.25)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
def test_peaked_scores_of_many_heads(torch, kvcache, bits, dim):
    # the same where whole steps are taken against an old maximum: late keys far above the ones before
    w = World(torch, kvcache, bits, "bf16", dim, 12, 64, [1400], [100], share=4.0)
    for pool in (0, 1):  # keys 900 .. 931 three times as large
        pages = w.table[0, torch.arange(900, 932) // 64].long()
        at = torch.arange(900, 932) % 64
        if bits == 16:
            p = w.pools[pool].cpu()
            p[pages, :, at] = p[pages, :, at] * 3
            w.pools[pool].copy_(p)
            w.held[0][pool][900:932] = p[pages, :, at].double()
        else:
            sc = w.scales[pool].cpu()
            sc[pages, :, at] = sc[pages, :, at] * 3
            w.scales[pool].copy_(sc)
            w.held[0][pool][900:932] = values(torch, w.pools[pool].cpu()[pages, :, at], sc[pages, :, at])
    check(torch, w, "bf16", 12, scale=0.25)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,kv", [(1, 2), (3, 2), (150, 2), (150, 16)])
def test_strides_and_alignment(torch, kvcache, bits, new, kv):
    # q as a block of a wider row, then one whose rows and heads start off 16-byte boundaries; out the same way
    heads = 3 * kv
    w = World(torch, kvcache, bits, "bf16", 64, kv, 64, [400, 151], [new, new])
    g = torch.Generator().manual_seed(5)
    q = torch.randn((w.tokens, heads, 64), generator=g).to(w.dt)
    exp = w.expect(q, 100, 2)
    for pad, off in ((64, 64), (3, 1)):
        wide = torch.full((w.tokens, heads, 64 + pad), float("nan"), dtype=w.dt, device="cuda")
        view = wide[:, :, off:off + 64]
        view.copy_(q)
        out_wide = torch.full_like(wide, 7.0)
        out = out_wide[:, :, off:off + 64]
        got = w.cache.attention(w.step(), view, window=100, sinks=2, out=out)
        sync()
        assert got is out
        assert float((out.cpu().double() - exp).abs().max()) <= bar(w, "bf16")
        out_wide[:, :, off:off + 64] = 7.0
        assert bool((out_wide == 7.0).all())  # nothing beside the rows was written


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv", [(1, 2), (4, 2), (200, 2), (200, 24)])
def test_hidden_values_stay_out(torch, kvcache, bits, dim, new, kv):
    # NaN and infinities in keys and values that a token does not see: those after it, those that its window has left
    # behind (their whole pages gone from the table too), and none of them in its output
    w = World(torch, kvcache, bits, "fp16", dim, kv, 64, [700], [new])
    heads, window, sinks = 2 * kv, 90, 70
    first = 700 - new + 1 - window  # the first key that any token sees past the sinks
    for t, fill in ((w.pools, float("nan")), (w.pools, float("inf"))):
        for which in range(2):
            for j in [70, 75, first - 1]:
                page, row = int(w.table[0, j // 64]), j % 64
                (w.pools if bits == 16 else w.scales)[which][page, :, row] = fill
        table = w.table.clone()
        for page in range(2, first // 64):
            w.table[0, page] = -1
        check(torch, w, "fp16", heads, window, sinks)
        w.table = table
    if new > 1:  # a NaN value of the last token reaches that token alone
        page, row = int(w.table[0, 699 // 64]), 699 % 64
        if bits == 16:
            w.pools[1][page, :, row, 3] = float("nan")
        else:
            w.scales[1][page, :, row, 0] = float("nan")
        g = torch.Generator().manual_seed(1)
        q = torch.randn((w.tokens, heads, dim), generator=g).to(w.dt)
        got = w.cache.attention(w.step(), q.cuda(), window=window, sinks=sinks)
        sync()
        got = got.cpu().double()
        exp = w.expect(q, window, sinks)
        assert float((got[:-1] - exp[:-1]).abs().max()) <= bar(w, "fp16")
        assert bool(got[-1, :, 3].isnan().all())


def test_pool_offsets_past_32_bits(torch, kvcache):
    # 2^31 and more elements before the pages in use
    for bits in (16, 4):
        w = World(torch, kvcache, bits, "bf16", 128, 8, 64, [200, 90], [1, 90], spare=0)
        pages = 70000 if bits == 16 else 140000
        big = [torch.empty((pages, *p.shape[1:]), dtype=p.dtype, device="cuda") for p in w.pools]
        bsc = [None if s is None else torch.empty((pages, *s.shape[1:]), dtype=s.dtype, device="cuda") for s in w.scales]
        n = w.pools[0].shape[0]
        assert big[0][:-n].numel() > 2 ** 31 if bits == 16 else big[0][:-n].numel() * 2 > 2 ** 31
        for b, p in zip(big + bsc, w.pools + w.scales):
            if b is not None:
                b[-n:] = p
        w.cache = kvcache.PagedCache.over(*big, *bsc)
        w.table = torch.where(w.table >= 0, w.table + pages - n, w.table)
        check(torch, w, "bf16", 16)
        k, v = w.cache.read(w.step(), w.tokens)
        sync()
        assert torch.equal(k.cpu().double(), torch.cat([h[0][-m:] for h, m in zip(w.held, w.news)]))
        assert torch.equal(v.cpu().double(), torch.cat([h[1][-m:] for h, m in zip(w.held, w.news)]))
        del big, bsc, w, k, v
        torch.cuda.empty_cache()


def rotate(torch, x, table, at, pairs):
    x = x.double()
    half = x.shape[-1] // 2
    y = x.clone()
    c = table[at].double()[:, None, :pairs]
    s = table[at].double()[:, None, half:half + pairs]
    y[..., :pairs] = x[..., :pairs] * c - x[..., half:half + pairs] * s
    y[..., half:half + pairs] = x[..., half:half + pairs] * c + x[..., :pairs] * s
    return y


def near_rounded(torch, got, exp, x, dtype):
    """got is exp rounded to the type, up to the FP32 arithmetic before it."""
    slack = 2.0 ** -22 * 2 * float(x.abs().max())
    nearest = exp.to(dtype_of(torch, dtype)).double()
    return bool(((got.double() - exp).abs() <= (nearest - exp).abs() + slack).all())


@pytest.mark.parametrize("dim,pairs", [(64, 32), (64, 16), (64, 5), (128, 64), (128, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lengths,news", [([1], [1]), ([5, 64, 65, 9], [1, 1, 1, 1]),
                                          ([33, 0, 150, 17, 20], [33, 0, 7, 1, 20]), ([4, 90], [9, 90])])
def test_append(torch, kvcache, lengths, news, bits, dtype, dim, pairs):
    heads, kv = 6, 2
    w = World(torch, kvcache, bits, dtype, dim, kv, 32, lengths, news)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn((w.tokens, heads + 2 * kv, dim), generator=g).to(w.dt)
    table = kvcache.rope_table(200, dim, pairs or None)
    dev = qkv.cuda()
    q, k, v = dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:]
    before = [p.clone() for p in w.pools]
    ones = all(n == 1 for n in news)
    for start in ([True, False] if ones else [True]):
        got_q = w.cache.append(w.step(start), k, v, q=q, rope=table, pairs=pairs)
        sync()
        rows, at, keep = [], [], []
        for s, (n, length) in enumerate(zip(news, lengths)):
            for i in range(n):
                rows.append(s)
                at.append(length - n + i)
                keep.append(length - n + i >= 0)
        at, keep, rows = torch.tensor(at), torch.tensor(keep), torch.tensor(rows)
        tab = table.cpu()
        exp_q = rotate(torch, qkv[keep][:, :heads], tab, at[keep], pairs)
        exp_k = rotate(torch, qkv[keep][:, heads:heads + kv], tab, at[keep], pairs)
        exp_v = qkv[keep][:, heads + kv:].double()
        assert near_rounded(torch, got_q.cpu()[keep], exp_q, qkv, dtype)
        page = w.table[rows[keep], at[keep] // 32].long()
        slot = at[keep] % 32
        got = [p.cpu()[page, :, slot] for p in w.pools]
        if bits == 16:
            assert near_rounded(torch, got[0], exp_k, qkv, dtype)
            assert torch.equal(got[1].double(), exp_v)
        else:
            for which, exp in enumerate((exp_k, exp_v)):
                sc = w.scales[which].cpu()[page, :, slot]
                val = values(torch, got[which], sc)
                gr = exp.unflatten(-1, (-1, 32))
                lo, hi = gr.amin(-1), gr.amax(-1)
                assert bool(((sc[..., 0].double() - (hi - lo) / 15).abs() <= 2.0 ** -10 * (hi - lo) / 15 + 2.0 ** -24).all())
                assert bool(((sc[..., 1].double() - lo).abs() <= 2.0 ** -11 * lo.abs() + 2.0 ** -20).all())
                most = (sc[..., 0].double() / 2 + 2.0 ** -11 * (hi - lo) + 2.0 ** -11 * lo.abs() + 2.0 ** -20)[..., None]
                most = (most + 2.0 ** -11 * gr.abs()).flatten(-2)
                assert bool(((val - exp).abs() <= most).all())
        # the rest of the pools is as it was
        for p, b in zip(w.pools, before):
            q_, b_ = p.cpu().clone(), b.cpu().clone()
            q_[page, :, slot] = 0
            b_[page, :, slot] = 0
            assert torch.equal(q_.view(torch.uint8), b_.view(torch.uint8))
        # and reads back as it stands
        rk, rv = w.cache.read(w.step(start), w.tokens)
        sync()
        if bits == 16:
            assert torch.equal(rk.cpu()[keep], got[0]) and torch.equal(rv.cpu()[keep], got[1])
        else:
            assert torch.equal(rk.cpu()[keep].double(), values(torch, got[0], w.scales[0].cpu()[page, :, slot]))
        assert bool((rk.cpu()[~keep] == 0).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_append_positions_in_place_and_unaligned(torch, kvcache, bits):
    # positions of their own, q rotated in place, rows that start off 16-byte boundaries, no rotation at all
    w = World(torch, kvcache, bits, "fp16", 64, 2, 16, [40, 21], [10, 21])
    g = torch.Generator().manual_seed(3)
    flat = torch.randn((w.tokens, 8 * 65 + 1), generator=g).to(w.dt)
    dev = flat.cuda()[:, 1:].unflatten(1, (8, 65))[:, :, :64]
    host = flat[:, 1:].unflatten(1, (8, 65))[:, :, :64]
    table = kvcache.rope_table(50, 64)
    at = torch.randint(0, 50, (w.tokens,), generator=g, dtype=torch.int32)
    q = dev[:, :4]
    got = w.cache.append(w.step(), dev[:, 4:6], dev[:, 6:8], q=q, rope=table, positions=at.cuda(), q_out=q)
    sync()
    assert got is q
    assert near_rounded(torch, q.cpu(), rotate(torch, host[:, :4], table.cpu(), at.long(), 32), flat, "fp16")
    k, v = w.cache.read(w.step(), w.tokens)
    exp = rotate(torch, host[:, 4:6], table.cpu(), at.long(), 32)
    step = 1.0 if bits == 4 else 0.0  # 4 bits: checked to their step above; here that the right rows arrived
    assert float((k.cpu().double() - exp).abs().max()) <= 0.3 * step + 0.01
    w.cache.append(w.step(), dev[:, 4:6], dev[:, 6:8])
    k, v = w.cache.read(w.step(), w.tokens)
    sync()
    if bits == 16:
        assert torch.equal(k.cpu(), host[:, 4:6]) and torch.equal(v.cpu(), host[:, 6:8])
    else:
        codes, sc = quantise(torch, host[:, 6:8])
        assert float((v.cpu().double() - values(torch, codes, sc)).abs().max()) <= 0.3


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_four_bit_codes_are_the_nearest(torch, kvcache, dim, dtype):
    # values on a 16-bit grid lie half way between two codes now and then: ties go to the even code, as in 64 bits. The
    # differences from the minimum are exact in FP32, and their quotient by the scale rounds to a tie only if it is one
    # (a quotient of two such numbers that is not a tie is further from it than FP32's rounding).
    w = World(torch, kvcache, 4, dtype, dim, 3, 32, [900], [900])
    g = torch.Generator().manual_seed(13)
    x = (torch.randn((900, 3, dim), generator=g) * 2).to(w.dt)
    w.cache.append(w.step(), x.cuda(), x.cuda())
    sync()
    at = torch.arange(900)
    page = w.table[0, at // 32].long()
    codes, scales = quantise(torch, x)
    for pool, sc in zip(w.pools, w.scales):
        assert torch.equal(sc.cpu()[page, :, at % 32], scales)
        assert torch.equal(pool.cpu()[page, :, at % 32], codes)


def test_four_bit_edges(torch, kvcache):
    # constant groups, zeros, subnormal ranges, values past FP16's range, infinities and a NaN
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    rows = []
    for fill in range(6):
        y = x.clone()
        if fill == 1:
            y[...] = 3.25
        elif fill == 2:
            y[..., 1] = 1e-7
        elif fill == 3:
            y[..., 0], y[..., 1] = 1e38, -1e38
        elif fill == 4:
            y[..., 0] = float("inf")
        elif fill == 5:
            y[..., 40] = float("nan")
        rows.append(y)
    k = torch.cat(rows).cuda()
    cache = kvcache.PagedCache(1, 16, 1, 64, bits=4)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    step = kvcache.Step(i32([6]), i32([[0]]), 6, i32([0, 6]), 6)
    cache.append(step, k, k)
    got, _ = cache.read(step, 6)
    sync()
    got = got.cpu().float()[:, 0]
    assert bool((got[0] == 0).all()) and bool((got[1] == 3.25).all())
    assert bool((got[2].abs() <= 1e-7).all())
    # FP16 has no scale that takes 15 steps from -65504 nearer to 65504: steps of 8, of which 15 stay 32 short
    assert 0 <= 65504 - float(got[3, 0]) <= 15 * 8 + 32 + 16 and float(got[3, 1]) == -65504
    assert float(got[4, 0]) == pytest.approx(65504, rel=1e-3) and float(got[4, 1]) == 0
    assert bool(got[5, 32:].isnan().all()) and bool((got[5, :32] == 0).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_large_and_small_queries(torch, kvcache, bits):
    # BF16 queries beyond FP16's range and far below it keep their scores (a 4-bit cache works in FP16 inside)
    w = World(torch, kvcache, bits, "bf16", 64, 1, 64, [300], [2])
    g = torch.Generator().manual_seed(2)
    base = torch.randn((2, 2, 64), generator=g)
    for size in (2.0 ** 20, 2.0 ** -30):
        q = (base * size).to(w.dt)
        got = w.cache.attention(w.step(), q.cuda(), scale=0.125 / size)
        sync()
        exp = w.expect(q, 0, 0, 0.125 / size)
        assert float((got.cpu().double() - exp).abs().max()) <= bar(w, "bf16")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,kv", [(1, 2), (200, 2), (200, 16)])
def test_streams_and_graphs(torch, kvcache, bits, new, kv):
    w = World(torch, kvcache, bits, "fp16", 64, kv, 64, [9000, 200], [new, new])
    g = torch.Generator().manual_seed(4)
    q = torch.randn((w.tokens, 2 * kv, 64), generator=g).to(w.dt)
    exp = w.cache.attention(w.step(), q.cuda())
    sync()
    side = torch.cuda.Stream()
    step, dev = w.step(), q.cuda()
    torch.cuda.synchronize()
    outs = []
    for k in range(4):  # two streams at once
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            outs.append(w.cache.attention(step, dev))
    torch.cuda.synchronize()
    assert all(torch.equal(o, exp) for o in outs)
    out = torch.empty_like(dev)
    graph = torch.cuda.CUDAGraph()
    live = torch.zeros_like(dev)
    with torch.cuda.graph(graph):
        w.cache.attention(step, live, out=out)
    live.copy_(dev)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, exp)
    del graph


def test_steps_outside_their_bounds_are_reported(torch, kvcache):
    # device arrays that break the call's bounds: no write, an error at the next sync, and the library usable after it
    w = World(torch, kvcache, 16, "fp16", 64, 2, 32, [64, 64], [2, 3])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    q = torch.zeros((5, 2, 64), dtype=w.dt).cuda()
    good = dict(length=[64, 64], table=w.table.tolist(), start=[0, 2, 5], max_length=64, max_new=3)
    bad = [dict(length=[64, 65]), dict(length=[-1, 64]), dict(start=[0, 2, 6]), dict(start=[0, 5, 5]),
           dict(start=[0, 3, 2]), dict(start=[-1, 2, 5]), dict(table=[w.table[0].tolist(), [99999, -5]]),
           dict(max_length=2000, length=[64, 1000])]
    for change in bad:
        c = {**good, **change}
        step = kvcache.Step(i32(c["length"]), i32(c["table"]), c["max_length"], i32(c["start"]), c["max_new"])
        before = [p.clone() for p in w.pools]
        for call in ("append", "attention", "read"):
            if call == "append":
                w.cache.append(step, q, q)
            elif call == "attention":
                w.cache.attention(step, q)
            else:
                w.cache.read(step, 5)
            with pytest.raises(_lib.JcArgumentError):
                sync()
        if "table" in change:  # the good sequence's rows were appended
            for p, b in zip(w.pools, before):
                p.copy_(b)
        else:
            n = sum(int(not torch.equal(p.view(torch.int16), b.view(torch.int16))) for p, b in zip(w.pools, before))
            assert n in (0, 2)
            for p, b in zip(w.pools, before):
                p.copy_(b)
    # a position outside the rotation table
    with pytest.raises(_lib.JcArgumentError):
        w.cache.append(w.step(), q, q, rope=kvcache.rope_table(62, 64))
        sync()
    sync()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,kv", [(1, 2), (90, 2), (90, 32)])
def test_a_page_outside_the_pool_is_left_out(torch, kvcache, bits, new, kv):
    w = World(torch, kvcache, bits, "fp16", 64, kv, 32, [200, 150], [new, new])
    g = torch.Generator().manual_seed(4)
    q = torch.randn((w.tokens, kv, 64), generator=g).to(w.dt)
    exp = w.expect(q, 0, 0)
    w.table[1, 1] = 10 ** 6
    got = w.cache.attention(w.step(), q.cuda())
    with pytest.raises(_lib.JcArgumentError):
        sync()
    assert float((got.cpu().double() - exp)[:new].abs().max()) <= bar(w, "fp16")  # the other sequence
    held = w.held[1]
    keep = [j for j in range(150) if not 32 <= j < 64]
    for i in (0, new - 1):  # without the page's keys
        at = 150 - new + i
        j = torch.tensor([x for x in keep if x <= at])
        z = torch.einsum("hd,jhd->hj", q[new + i].double(), held[0][j]) * 0.125
        o = torch.einsum("hj,jhd->hd", torch.softmax(z, -1), held[1][j])
        assert float((got[new + i].cpu().double() - o).abs().max()) <= bar(w, "fp16")


def test_refusals(torch, kvcache):
    cache = kvcache.PagedCache(4, 32, 2, 64, dtype=torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    step = kvcache.Step(i32([5, 6]), i32([[0], [1]]), 6)
    x = torch.zeros((2, 2, 64), dtype=torch.float16).cuda()
    ok = cache.append(step, x, x, q=x)
    assert ok.shape == x.shape
    bad = [lambda: cache.append(step, x.bfloat16(), x.bfloat16()), lambda: cache.append(step, x, x.bfloat16()),
           lambda: cache.append(step, x[:, :1], x), lambda: cache.append(step, x[:1], x[:1]),
           lambda: cache.append(step, x.cpu(), x.cpu()), lambda: cache.append(step, x, x, q_out=x),
           lambda: cache.append(step, x, x, rope=torch.zeros((4, 32)).cuda()),
           lambda: cache.append(step, x, x, rope=torch.zeros((9, 64)).cuda(), pairs=33),
           lambda: cache.append(step, x, x, positions=torch.zeros(2).cuda()),
           lambda: cache.append(step, x, x, q=x, q_out=x[:1].expand(2, 2, 64)),
           lambda: cache.attention(step, x[:, :, ::2]), lambda: cache.attention(step, x[:, :1]),
           lambda: cache.attention(step, x, window=-1), lambda: cache.attention(step, x, sinks=-1),
           lambda: cache.attention(step, x, scale=0.0), lambda: cache.attention(step, x, scale=float("nan")),
           lambda: cache.attention(step, x.float()), lambda: cache.attention(step, x, out=x.bfloat16()),
           lambda: cache.attention(step, x, out=x[:1]), lambda: cache.attention(step, torch.cat([x, x])),
           lambda: kvcache.Step(i32([5]), i32([[0], [1]]), 6), lambda: kvcache.Step(i32([5]), i32([[0]]), -1),
           lambda: kvcache.Step(i32([5]), i32([[0]]), 6, i32([0]), 1), lambda: kvcache.Step(i32([5]), i32([[0]]), 6, None, 2),
           lambda: kvcache.Step(i32([5]).long(), i32([[0]]), 6), lambda: kvcache.Step(i32([5]).cpu(), i32([[0]]), 6),
           lambda: kvcache.PagedCache(4, 32, 2, 64, bits=8), lambda: kvcache.PagedCache(4, 32, 2, 64, torch.float16, 4),
           lambda: kvcache.PagedCache.over(cache.k, cache.v[:2]), lambda: kvcache.PagedCache.over(cache.k.float(), cache.v.float()),
           lambda: kvcache.PagedCache.over(cache.k.view(torch.uint8), cache.v.view(torch.uint8)),
           lambda: kvcache.PagedCache.over(cache.k.transpose(1, 2), cache.v.transpose(1, 2))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} was not one")
    for page, dim in ((20, 64), (8, 64), (32, 96)):
        c = kvcache.PagedCache(4, page, 2, dim, dtype=torch.float16)
        with pytest.raises(_lib.JcArgumentError):
            c.attention(step, torch.zeros((2, 2, dim), dtype=torch.float16).cuda())
    sync()


def test_no_tokens_and_no_sequences(torch, kvcache):
    cache = kvcache.PagedCache(4, 32, 2, 64, dtype=torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    x = torch.zeros((0, 2, 64), dtype=torch.float16).cuda()
    none = kvcache.Step(i32([]), i32([]).view(0, 1), 0)
    empty = kvcache.Step(i32([3]), i32([[0]]), 3, i32([0, 0]), 0)
    for step in (none, empty):
        assert cache.append(step, x, x, q=x).shape == (0, 2, 64)
        assert cache.attention(step, x).shape == (0, 2, 64)
        assert cache.read(step, 0)[0].shape == (0, 2, 64)
    sync()


@pytest.mark.parametrize("partial", [1.0, 0.5])
def test_streamed_patches_match_the_time_attention_of_the_whole_series(torch, kvcache, partial):
    # a Timestral layer's time attention (all patches observed) token by token over a cache, against
    # jc_time_attention_device on the whole rows: two separate kernels of FP16 rounding each, so twice the bar
    rows, n, heads = 3, 130, 4
    d = heads * 64
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn((rows, n, 3, heads, 64), generator=g).half().cuda()
    pairs = int(32 * partial)
    table = kvcache.rope_table(n, 64, pairs)
    cache = kvcache.PagedCache(rows * 3, 64, heads, 64, dtype=torch.float16)
    pages = torch.arange(rows * 3, dtype=torch.int32).view(rows, 3).flip(1).contiguous().cuda()
    length = torch.zeros(rows, dtype=torch.int32, device="cuda")
    got, rot = [], []
    done = 0
    for new in (100, 1, 1, 20, 1, 7):  # a prompt, then patches as they arrive
        length += new
        done += new
        start = torch.arange(0, (rows + 1) * new, new, dtype=torch.int32, device="cuda")
        step = kvcache.Step(length, pages, n, start, new)
        part = qkv[:, done - new:done].reshape(rows * new, 3, heads, 64)
        q = cache.append(step, part[:, 1], part[:, 2], q=part[:, 0], rope=table, pairs=pairs)
        got.append(cache.attention(step, q).view(rows, new, d))
        rot.append(q.view(rows, new, heads, 64))
    sync()
    assert done == n
    whole = kvcache.Step(length, pages, n, torch.arange(0, (rows + 1) * n, n, dtype=torch.int32, device="cuda"), n)
    k, v = cache.read(whole, rows * n)
    fused = torch.stack([torch.cat(rot, 1).view(rows * n, heads, 64), k, v], 1).contiguous()
    out = torch.empty((rows * n, d), dtype=torch.float16, device="cuda")
    ones = torch.ones(rows * n, dtype=torch.int32, device="cuda")
    zero = torch.zeros(rows, dtype=torch.int32, device="cuda")
    _lib.check(_lib.lib().jc_time_attention_device(
        0, _lib.FP16, fused.data_ptr(), 3 * d, None, 0, out.data_ptr(), d, rows, n, heads, 64, d, 0.125, 0, n, n,
        ones.data_ptr(), zero.data_ptr(), None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    sync()
    most = float(v.abs().max())
    err = float((torch.cat(got, 1).reshape(rows * n, d).double() - out.double()).abs().max())
    assert err <= 2 * (2 * ROUNDING["fp16"] + 1e-4) * most and math.isfinite(err)
