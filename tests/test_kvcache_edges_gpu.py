"""The paged cache's attention where its arithmetic or its arguments are at an edge, against the definition in 64 bits.

The bars are those of test_kvcache_gpu.py, whose cache of known contents these tests share.
"""

import math

import pytest
from test_kvcache_gpu import ROUNDING, World, bar, dtype_of, quantise, sync, values

from jitcast_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kvcache(jc):
    from jitcast_b200 import kvcache

    return kvcache


def put(torch, w, which, s, j, x):
    """Key (which 0) or value (1) of index j of sequence s becomes x [kv_heads, dim]: in the pools and in what they hold."""
    x = x.to(w.dt)
    page, row = int(w.table[s, j // w.page]), j % w.page
    if w.bits == 16:
        w.pools[which][page, :, row] = x.cuda()
        w.held[s][which][j] = x.double()
    else:
        codes, scales = quantise(torch, x)
        w.pools[which][page, :, row] = codes.cuda()
        w.scales[which][page, :, row] = scales.cuda()
        w.held[s][which][j] = values(torch, codes, scales)


def spoil(w, which, s, j, value=float("nan"), dim=5):
    """One dim (4 bits: its group of 32, which then reads as NaN) of index j becomes `value`."""
    page, row = int(w.table[s, j // w.page]), j % w.page
    if w.bits == 16:
        w.pools[which][page, :, row, dim] = value
        w.held[s][which][j, :, dim] = value
    else:
        w.scales[which][page, :, row, dim // 32] = float("nan")
        w.held[s][which][j, :, dim // 32 * 32:dim // 32 * 32 + 32] = float("nan")


def queries(torch, w, heads, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((w.tokens, heads, w.dim), generator=g).to(w.dt)


def agree(got, exp, most):
    """NaN exactly where the definition has one, the rest within the bar."""
    got = got.cpu().double()
    assert bool((got.isnan() == exp.isnan()).all())
    there = ~exp.isnan()
    assert not there.any() or float((got - exp)[there].abs().max()) <= most


# The forms that a call can take: (kv heads, lengths, new tokens). Whole rows by one block of the splits, rows joined from
# several, 256-row tiles, and tiles whose keys are split over CTAs and joined.
FORMS = {
    "splits": (2, [90, 1, 40], [2, 1, 1]),
    "joined splits": (2, [9000, 1, 40], [2, 1, 1]),
    "tiles": (8, [300, 1, 40], [150, 1, 3]),
    "joined tiles": (8, [4500, 1, 200], [70, 1, 45]),
}


@pytest.mark.parametrize("bits,dtype", [(16, "bf16"), (16, "fp16"), (4, "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_visible_nans_reach_the_output(torch, kvcache, form, dim, bits, dtype):
    # a NaN score makes its row's softmax NaN, wherever the key lies and whatever came before it
    kv, lengths, news = FORMS[form]
    heads = 2 * kv
    for what in ("query", "first key", "every key", "sink"):
        w = World(torch, kvcache, bits, dtype, dim, kv, 64, lengths, news)
        q = queries(torch, w, heads)
        window, sinks = (20, 3) if what == "sink" else (0, 0)
        if what == "query":
            q[0, 1, 7] = float("nan")
            q[w.bounds[1], heads - 1, 0] = float("nan")  # the sequence of one key
        elif what == "every key":
            for j in range(lengths[2]):
                spoil(w, 0, 2, j)
            spoil(w, 0, 1, 0)
        else:
            spoil(w, 0, 0, 0)
        got = w.cache.attention(w.step(), q.cuda(), window=window, sinks=sinks)
        sync()
        agree(got, w.expect(q, window, sinks), bar(w, dtype))


@pytest.mark.parametrize("bits,dtype", [(16, "fp16"), (16, "bf16"), (4, "fp16"), (4, "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 300, 37000])
def test_many_small_probabilities_keep_their_weight(torch, kvcache, new, dim, bits, dtype):
    # one key 18 above 131,000 others: each of them has a probability below FP16's smallest, 2^-25.97, and all together
    # 1/500 of the output. One row's and 300 rows' keys are split over CTAs, most of which never meet the large one; those of
    # 37,000 rows are not.
    n, dt = 131072, dtype_of(torch, dtype)
    pages = n // 1024
    key, value = torch.zeros((n, 1, dim)), torch.ones((n, 1, dim))
    key[0, 0, 0], value[0] = 2.25, 0.0
    pools, scales, first = [], [], None
    for x in (key, value):
        x = x.to(dt)
        if bits == 16:
            pools.append(x.view(pages, 1024, 1, dim).transpose(1, 2).contiguous().cuda())
            scales.append(None)
            first = float(x[0, 0, 0]) if first is None else first
        else:
            c, s = quantise(torch, x)
            first = float(values(torch, c[:1], s[:1])[0, 0, 0]) if first is None else first
            pools.append(c.view(pages, 1024, 1, -1).transpose(1, 2).contiguous().cuda())
            scales.append(s.view(pages, 1024, 1, -1, 2).transpose(1, 2).contiguous().cuda())
    cache = kvcache.PagedCache.over(*pools, *scales)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    step = kvcache.Step(i32([n]), torch.arange(pages, dtype=torch.int32).view(1, -1).cuda(), n, i32([0, new]), new)
    q = torch.zeros((new, 1, dim), dtype=dt)
    q[..., 0] = 8.0
    got = cache.attention(step, q.cuda(), scale=1.0).cpu().double()
    sync()
    others = torch.arange(n - new, n, dtype=torch.float64)
    exp = (others / (others + math.exp(8.0 * first)))[:, None, None].expand_as(got)
    err = float((got - exp).abs().max())
    print(f"max error {err:.2e}, output {float(exp.max()):.2e}")
    assert err <= 2 * ROUNDING[dtype] + 1e-4  # the bar, with max |v| = 1


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_rows_of_infinitely_small_scores(torch, kvcache, form, dim, dtype):
    # every visible score -inf: the softmax is undefined (zeros are for a token that sees no key); some: they weigh nothing
    kv, lengths, news = FORMS[form]
    w = World(torch, kvcache, 16, dtype, dim, kv, 64, lengths, news)
    q = queries(torch, w, 2 * kv)
    q[:, :, 5] = q[:, :, 5].abs() + 1
    for j in range(lengths[2]):
        spoil(w, 0, 2, j, float("-inf"))
    spoil(w, 0, 1, 0, float("-inf"))
    spoil(w, 0, 0, 0, float("-inf"))
    got = w.cache.attention(w.step(), q.cuda())
    sync()
    exp = w.expect(q, 0, 0)
    assert exp[w.bounds[1]:].isnan().all() and not exp[:w.bounds[1]].isnan().any()
    agree(got, exp, bar(w, dtype))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,lengths,news", [(2, [90, 41], [3, 3]), (2, [9000, 41], [3, 3]), (8, [300, 70], [150, 3]),
                                             (8, [4500, 200], [70, 45])])
def test_out_may_be_q(torch, kvcache, kv, lengths, news, dim, bits):
    # in place, with a value that only the last token sees undefined, so that the rows before it are worked out again
    w = World(torch, kvcache, bits, "bf16", dim, kv, 64, lengths, news)
    spoil(w, 1, 0, lengths[0] - 1)
    spoil(w, 1, 1, lengths[1] - 1)
    q = queries(torch, w, 2 * kv)
    dev = q.cuda()
    got = w.cache.attention(w.step(), dev, out=dev)
    sync()
    assert got is dev
    agree(got, w.expect(q, 0, 0), bar(w, "bf16"))


@pytest.mark.parametrize("bits", [16, 4])
def test_an_undefined_value_does_not_stall_a_call(torch, kvcache, bits):
    # a value of the first key undefined: every row of the prompt is worked out again, key by key. A row's 4,096 keys one
    # after another at a memory latency each, 32 rows a warp, would take some 50 ms, a thousand times the call.
    n, kv = 4096, 4
    w = World(torch, kvcache, bits, "fp16", 64, kv, 64, [n], [n])
    q = queries(torch, w, kv).cuda()
    step, out = w.step(), torch.empty_like(q)

    def time():
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            w.cache.attention(step, q, out=out)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    clean = time()
    spoil(w, 1, 0, 0)
    redone = time()
    print(f"{clean:.3f} ms, with every row worked out again {redone:.3f} ms")
    assert bool(out[:, :, 5].isnan().all())
    assert redone < 100 * clean


def test_another_callers_product_does_not_take_a_cache_error(torch, kvcache, jc):
    import numpy as np

    w = World(torch, kvcache, 16, "fp16", 64, 2, 32, [64], [1])
    bad = kvcache.Step(torch.tensor([65], dtype=torch.int32).cuda(), w.table.cuda(), 64)
    q = torch.zeros((1, 2, 64), dtype=w.dt).cuda()
    w.cache.attention(bad, q)
    torch.cuda.synchronize()
    x = np.ones((4, 64), np.float32)
    y = jc.ops.linear(x, x, np.zeros(4, np.float32), precision="bf16")  # a right product
    assert (y == 64).all()
    with pytest.raises(_lib.JcArgumentError):  # and the cache's caller hears of its own error
        sync()
    sync()


def test_a_steps_bounds_may_grow_and_its_tensors_stay(torch, kvcache):
    w = World(torch, kvcache, 16, "fp16", 64, 2, 32, [90], [1])
    q = queries(torch, w, 2)
    length = torch.tensor([40], dtype=torch.int32).cuda()
    step = kvcache.Step(length, w.table.cuda(), 40)
    w.cache.attention(step, q.cuda())
    sync()
    length.fill_(90)
    step.max_length = 90
    got = w.cache.attention(step, q.cuda())
    sync()
    assert float((got.cpu().double() - w.expect(q, 0, 0)).abs().max()) <= bar(w, "fp16")
    for change in (lambda: setattr(step, "max_length", -1), lambda: setattr(step, "max_new", 2)):
        with pytest.raises(ValueError):
            change()
    assert (step.max_length, step.max_new) == (90, 1)
    # what a call reads stays what it was made of
    for change in (lambda: setattr(step, "length", length.clone()), lambda: setattr(step, "page_table", w.table.cuda()),
                   lambda: setattr(step, "start", length), lambda: setattr(w.cache, "k", w.cache.k.clone()),
                   lambda: setattr(w.cache, "v_scale", None)):
        with pytest.raises(AttributeError):
            change()


@pytest.mark.parametrize("new", [1, 3, 150])
def test_outputs_of_heads_before_tokens(torch, kvcache, new):
    # [heads, tokens, dim] tensors seen as [tokens, heads, dim]: rows that do not overlap, in the other order
    w = World(torch, kvcache, 16, "bf16", 64, 2, 64, [200], [new])
    q = queries(torch, w, 6)
    like = lambda x: x.cuda().transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    dev, out = like(q), like(torch.zeros_like(q))
    got = w.cache.attention(w.step(), dev, out=out)
    sync()
    assert got is out
    assert float((out.cpu().double() - w.expect(q, 0, 0)).abs().max()) <= bar(w, "bf16")
    k = queries(torch, w, 2, 3)
    out.zero_()
    w.cache.append(w.step(), like(k), like(k), q=dev, q_out=out)
    sync()
    assert torch.equal(out.cpu(), q)
    assert torch.equal(w.cache.read(w.step(), new)[0].cpu(), k)
