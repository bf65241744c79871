"""The serving operators over a paged key/value cache, as a user calls them, and their plain forms.

Three operators: appending new tokens' keys and values (position rotation on the way, cache in 16 or 4 bits),
attention with a sliding window and sinks over a 16-bit cache, and the same attention over a 4-bit cache.

A cache is a pool of pages. 16 bits: k, v [pages, kv_heads, page, dim]. 4 bits: codes [pages, kv_heads, page,
dim / 2] (byte j holds dim 2j in its low half, 2j + 1 in its high half) and, per 32 dims, a pair (scale, min) in
FP16 [pages, kv_heads, page, dim / 32, 2]; a code stands for fp16(code * scale + min).
A step has, per sequence, its cached length (new tokens included), its pages in order, and its new tokens, packed
over the sequences (`start` has the bounds). A new token's index t is its place in its sequence; it sees the keys
j <= t with j > t - window or j < sinks (window 0: all).
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32   # dims that share a 4-bit scale
BLOCK = 128  # queries that share one gathered key list in the plain form


# ---- cases ---------------------------------------------------------------------------------------------------------

def _case(name, op, type, bits, seqs, new, length, heads, kv_heads, dim, page, window=0, sinks=0, pairs=0):
    """`new` and `length` are [least, most] over the sequences; a sequence's length has its new tokens in it."""
    return {"name": name, "op": op, "type": type, "bits": bits, "seqs": seqs, "new_lo": new[0], "new_hi": new[1],
            "len_lo": length[0], "len_hi": length[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window, "sinks": sinks, "pairs": pairs}


def listed():
    return [
        # one new patch of a few series in a rolling forecast, half of each head rotating: pure latency
        _case("append 8 series, one token", "append", "bf16", 16, 8, (1, 1), (90, 700), 16, 16, 64, 64, pairs=16),
        # the histories of new series enter the cache, ragged, all layers' width at once
        _case("append 7 prompts", "append", "bf16", 16, 7, (900, 4100), (900, 4100), 16, 16, 64, 64, pairs=16),
        # prompt chunks into a 4-bit cache with shared key heads, and the cached tokens read back
        _case("append 37 chunks, 4 bits", "append", "fp16", 4, 37, (60, 420), (100, 900), 32, 8, 128, 32, pairs=64),
        # the smallest attention call: one new patch of four short series
        _case("window, 4 series, one token", "attention", "fp16", 16, 4, (1, 1), (190, 400), 16, 16, 64, 64, 128, 4),
        # a serving batch of long histories, one token each, grouped heads, window and sinks
        _case("window, 96 series, one token", "attention", "bf16", 16, 96, (1, 1), (2100, 20000), 32, 8, 128, 64,
              4096, 16),
        # first pass over many short series: 128 patches of context and two forecast tokens each
        _case("window, 64 series of 130", "attention", "fp16", 16, 64, (130, 130), (130, 130), 16, 16, 64, 64),
        # first pass over two long histories with a window and sinks
        _case("window, 2 long prompts", "attention", "bf16", 16, 2, (11003, 12800), (11003, 12800), 16, 16, 64, 64,
              2048, 64),
        # chunks of prompts over longer contexts, every key visible, wide grouped heads
        _case("window off, 3 chunks", "attention", "bf16", 16, 3, (501, 1500), (3001, 9000), 32, 8, 128, 128),
        # 4 bits: the smallest call
        _case("4 bits, 3 series, one token", "attention", "bf16", 4, 3, (1, 1), (350, 611), 16, 16, 64, 64),
        # 4 bits: a serving batch whose cache would not be small in 16 bits
        _case("4 bits, 48 series, one token", "attention", "bf16", 4, 48, (1, 1), (5000, 32500), 32, 8, 128, 64),
        # 4 bits: one very long history, two tokens, alone on the GPU
        _case("4 bits, one long series", "attention", "fp16", 4, 1, (2, 2), (131231, 131231), 16, 16, 64, 16),
        # 4 bits: chunks of prompts with a window and sinks
        _case("4 bits, 4 chunks", "attention", "bf16", 4, 4, (200, 411), (2500, 6100), 32, 8, 128, 64, 2000, 8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["append", "append", "one", "one", "prompt"])
        bits = rng.choice([16, 4])
        dim = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
        page = rng.choice([16, 32, 48, 64, 128])
        seqs = _log(rng, 1, 100)
        if kind == "one":
            new = _log(rng, 1, 3)
            new = (new, new)
            hi = _log(rng, 20, 40000)
        else:
            hi = _log(rng, 20, 12000)
            new = (max(1, hi // rng.randint(4, 60)), max(1, hi // rng.choice([1, 2, 3])))
        lo = max(new[1], hi // rng.randint(1, 9))
        hi = max(lo, hi)
        window = rng.choice([0, _log(rng, 16, 8000)])
        c = _case("", "append" if kind == "append" else "attention", rng.choice(["bf16", "fp16"]), bits, seqs, new,
                  (lo, hi), heads, kv, dim, page, 0 if kind == "append" else window,
                  0 if kind == "append" or not window else rng.choice([0, 1, 4, _log(rng, 1, 150)]),
                  rng.choice([dim // 4, dim // 2]) if kind == "append" else 0)
        del c["name"]
        shapes = (heads, kv, heads * dim, kv * dim, 2 * (heads + kv) * dim, (heads + 2 * kv) * dim, lo, hi, new[0], new[1], window, sum(_news(c)))
        if heads <= 64 and 3072 not in shapes and _cost(c) <= most and _room(c) <= 6e9:
            return c


def _spread(lo, hi, n, turn):
    """n whole numbers from lo to hi, both ends among them, in a mixed order that `turn` sets."""
    if n == 1:
        return [hi]
    return [lo + ((hi - lo) * ((i * 7 + turn) % n)) // (n - 1) if n % 7 else lo + ((hi - lo) * ((i * 5 + turn) % n)) // (n - 1)
            for i in range(n)]


def _news(case):
    return [min(a, b) for a, b in zip(_spread(case["new_lo"], case["new_hi"], case["seqs"], 0), _lengths(case))]


def _lengths(case):
    n = case["seqs"]
    if (case["new_lo"], case["new_hi"]) == (case["len_lo"], case["len_hi"]):
        return _spread(case["len_lo"], case["len_hi"], n, 0)  # whole prompts: no context before the new tokens
    return _spread(case["len_lo"], case["len_hi"], n, 3)


def _seen(case):
    """(visible pairs, keys that some query sees), summed over the sequences."""
    w, s, pairs, keys = case["window"], case["sinks"], 0, 0
    for n, L in zip(_news(case), _lengths(case)):
        t = np.arange(L - n, L, dtype=np.int64)
        band = t + 1 if w == 0 else np.minimum(t + 1, w)
        pairs += int((band + np.minimum(s, t + 1 - band)).sum())
        first = int(t[0] + 1 - band[0])
        keys += L - first + min(s, first)
    return pairs, keys


def work(case):
    size, D, tokens = 2, case["dim"], sum(_news(case))
    slot = D * size if case["bits"] == 16 else D // 2 + D // GROUP * 4  # one token's key (or value) of one head
    if case["op"] == "append":
        rows = tokens * (case["heads"] + 2 * case["kv_heads"])
        b = rows * D * size + tokens * case["heads"] * D * size + 2 * tokens * case["kv_heads"] * slot
        b += tokens * case["pairs"] * 2 * 4
        f = 6 * tokens * (case["heads"] + case["kv_heads"]) * case["pairs"]
        if case["bits"] == 4:  # and the sequences read back
            b += 2 * sum(_lengths(case)) * case["kv_heads"] * (slot + D * size)
            f += 4 * 2 * tokens * case["kv_heads"] * D + 2 * 2 * sum(_lengths(case)) * case["kv_heads"] * D
        return {"bytes": b, "flops": f}
    pairs, keys = _seen(case)
    return {"bytes": 2 * tokens * case["heads"] * D * size + 2 * keys * case["kv_heads"] * slot,
            "flops": 4 * pairs * case["heads"] * D}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def _room(case):
    """Bytes of the plain form's largest arrays: the gathered keys and the scores, in 32 bits."""
    new, length = max(_news(case)), max(_lengths(case))
    if case["op"] == "append":
        return 4 * sum(_news(case)) * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    items = case["seqs"] * -(-new // BLOCK)
    keys = _keys(case, new, length)
    return 4 * items * keys * (case["kv_heads"] * case["dim"] + case["heads"] * min(new, BLOCK))


def _keys(case, new, length):
    return min(length, case["sinks"] + case["window"] + min(new, BLOCK) - 1) if case["window"] else length


# ---- inputs --------------------------------------------------------------------------------------------------------

def _page_ids(case, rng):
    need = [-(-L // case["page"]) for L in _lengths(case)]
    ids = list(range(sum(need) + 3))  # a few pages stay free
    rng.shuffle(ids)  # a pool in use hands its pages out in no order
    table = np.full((case["seqs"], max(need)), -1, np.int32)
    for s, m in enumerate(need):
        table[s, :m] = ids[:m]
        del ids[:m]
    return sum(need) + 3, table


def _pool(gen, pages, case, offset):
    """A pool of normal values, about channel means of their own where `offset` (keys have them)."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    if offset:
        x += torch.randn((1, case["kv_heads"], 1, case["dim"]), generator=gen, device=DEV)
    return x


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    type = TYPES[case["type"]]
    D, H, G = case["dim"], case["heads"], case["kv_heads"]
    pages, table = _page_ids(case, rng)
    lengths, news = _lengths(case), _news(case)
    tokens = sum(news)
    st = dict(case=dict(case), tokens=tokens, max_len=max(lengths), max_new=max(news),
              length=torch.tensor(lengths, dtype=torch.int32, device=DEV),
              start=torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=DEV),
              table=torch.from_numpy(table).to(DEV), scales=(None, None))
    if case["bits"] == 16:
        st["k"], st["v"] = (_pool(gen, pages, case, key).to(type) for key in (True, False))
    else:
        (st["k"], ks), (st["v"], vs) = (_pack(_pool(gen, pages, case, key)) for key in (True, False))
        st["scales"] = (ks, vs)
    # the projections' output, as the models' q|k|v|gate product leaves it: one row a token
    qkv = torch.randn((tokens, 2 * H + 2 * G, D), generator=gen, device=DEV).to(type)
    st["q"], st["new_k"], st["new_v"] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:H + 2 * G]
    if case["op"] == "append":
        # cos and sin by position; a partial rotation has them for its pairs only
        at = np.arange(st["max_len"])[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))[None]
        st["rope"] = torch.tensor(np.concatenate([np.cos(at), np.sin(at)], 1), dtype=torch.float32, device=DEV)
    if case["op"] == "append" and case["bits"] == 4:
        # for the read-back: the sequences' whole lengths
        st["whole"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEV)
        st["whole_tokens"] = sum(lengths)
    if own:  # the handles that a serving loop keeps: the cache over its pools, the step's lengths and pages
        from jitcast_b200 import kvcache

        ks, vs = st["scales"]
        st["cache"] = kvcache.PagedCache.over(st["k"], st["v"], ks, vs)
        one = st["max_new"] == 1
        st["step"] = kvcache.Step(st["length"], st["table"], st["max_len"], None if one else st["start"], st["max_new"])
        if "whole" in st:
            st["all"] = kvcache.Step(st["length"], st["table"], st["max_len"], st["whole"], st["max_len"])
    return st


# ---- the operators -------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if case["op"] == "append":
        return _append_own(st) if own else _append_plain(st)
    if own:
        return st["cache"].attention(st["step"], st["q"], window=case["window"], sinks=case["sinks"])
    return _attention_plain(st)


def _append_own(st):
    case, cache = st["case"], st["cache"]
    q = cache.append(st["step"], st["new_k"], st["new_v"], q=st["q"], rope=st["rope"], pairs=case["pairs"])
    if case["bits"] == 16:
        return {"q": q, "k": st["k"], "v": st["v"]}
    k, v = cache.read(st["all"], st["whole_tokens"])
    return {"q": q, "k": k, "v": v}


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _pack(x):
    """(codes, scales) of 32-bit values x [..., dim]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    scale, low = ((hi - lo) / 15).half(), lo.half()
    s, m = scale.float()[..., None], low.float()[..., None]
    codes = torch.where(s > 0, (g - m) / s, 0).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack([scale, low], -1)


def _unpack(codes, scales):
    """The values, in 32 bits, that packed codes [..., dim / 2] stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    s = scales.float()
    return (c * s[..., :1] + s[..., 1:]).flatten(-2).half().float()


def _rotate(x, rope, at, pairs):
    """x [tokens, heads, dim] in 32 bits, rotated by its tokens' positions `at`."""
    x = x.float()
    half = x.shape[-1] // 2
    c, s = rope[at][:, None, :pairs], rope[at][:, None, half:half + pairs]
    a, b = x[..., :pairs], x[..., half:half + pairs]
    return torch.cat([a * c - b * s, x[..., pairs:half], b * c + a * s, x[..., half + pairs:]], -1)


def _places(st, start, tokens):
    """(sequence, index in it) of each packed token."""
    t = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), t.int(), right=True)
    return seq, st["length"][seq].long() - start[seq + 1] + t


def _append_plain(st):
    case, page = st["case"], st["case"]["page"]
    seq, at = _places(st, st["start"], st["tokens"])
    ids, row = st["table"][seq, at // page].long(), at % page
    type = st["q"].dtype
    q = _rotate(st["q"], st["rope"], at, case["pairs"]).to(type)
    k, v = _rotate(st["new_k"], st["rope"], at, case["pairs"]), st["new_v"]
    if case["bits"] == 16:
        st["k"][ids, :, row] = k.to(type)
        st["v"][ids, :, row] = v
        return {"q": q, "k": st["k"], "v": st["v"]}
    ks, vs = st["scales"]
    st["k"][ids, :, row], ks[ids, :, row] = _pack(k)
    st["v"][ids, :, row], vs[ids, :, row] = _pack(v)
    seq, at = _places(st, st["whole"], st["whole_tokens"])
    ids, row = st["table"][seq, at // page].long(), at % page
    return {"q": q, "k": _unpack(st["k"][ids, :, row], ks[ids, :, row]).half(),
            "v": _unpack(st["v"][ids, :, row], vs[ids, :, row]).half()}


def _attention_plain(st):
    """Queries in blocks; each block gathers the keys that any of its queries may see (the sinks, then the band)."""
    case = st["case"]
    n, H, G, D, page = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    window, sinks = case["window"], case["sinks"]
    B = min(st["max_new"], BLOCK)
    blocks = -(-st["max_new"] // B)
    length, start = st["length"].long(), st["start"].long()
    new = start[1:] - start[:-1]
    # [sequence, block, query]: its place among the new tokens, its packed row and its index t in the sequence
    i = torch.arange(blocks * B, device=DEV).view(1, blocks, B).expand(n, -1, -1)
    there = i < new[:, None, None]
    row = torch.where(there, start[:-1, None, None] + i, 0)
    t = (length - new)[:, None, None] + i
    # [sequence, block, key]: the gathered keys' indexes
    keys = _keys(case, st["max_new"], st["max_len"])
    j = torch.arange(keys, device=DEV).expand(n, blocks, -1)
    if window:
        band = (t[:, :, :1] - window + 1 - sinks).clamp(min=0)
        j = torch.where(j < sinks, j, j + band)
    held = j < length[:, None, None]
    jj = torch.where(held, j, 0)
    ids = st["table"][torch.arange(n, device=DEV)[:, None, None], jj // page].long()
    k, v = st["k"][ids, :, jj % page], st["v"][ids, :, jj % page]  # [sequence, block, key, kv head, ..]
    if case["bits"] == 4:
        ks, vs = st["scales"]
        k, v = _unpack(k, ks[ids, :, jj % page]), _unpack(v, vs[ids, :, jj % page])
    q = st["q"][row].float().unflatten(3, (G, H // G))  # [sequence, block, query, kv head, group, dim]
    s = torch.einsum("nbqgrd,nbkgd->nbgrqk", q, k.float()) / math.sqrt(D)
    see = held[:, :, None] & (j[:, :, None] <= t[..., None])
    if window:
        see = see & ((j[:, :, None] > t[..., None] - window) | (j[:, :, None] < sinks))
    s = s.masked_fill(~see[:, :, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.einsum("nbgrqk,nbkgd->nbqgrd", p, v.float())
    return o.flatten(3, 4)[there].to(st["q"].dtype)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _values64(code, pair):
    """What codes [.., dim / 2] with pairs [.., dim / 32, 2] stand for."""
    c = torch.empty((*code.shape[:-1], code.shape[-1] * 2), dtype=torch.float64, device=DEV)
    c[..., 0::2] = (code % 16).double()
    c[..., 1::2] = (code // 16).double()
    scale = pair[..., 0].double().repeat_interleave(GROUP, -1)
    low = pair[..., 1].double().repeat_interleave(GROUP, -1)
    return (low + scale * c).half().double()


def _codes64(x):
    """x [.., dim] in 64 bits -> the values that its 4-bit form stands for."""
    parts = []
    for g in range(x.shape[-1] // GROUP):
        y = x[..., g * GROUP:(g + 1) * GROUP]
        low = y.min(-1, keepdim=True).values
        scale = ((y.max(-1, keepdim=True).values - low) / 15).half().double()
        low = low.half().double()
        code = torch.round((y - low) / torch.where(scale > 0, scale, 1)).clamp(0, 15)
        parts.append((low + code * torch.where(scale > 0, scale, 0)).half().double())
    return torch.cat(parts, -1)


def exact(case, seed):
    st = prepare(case, seed)
    D, page = case["dim"], case["page"]
    lengths, news = _lengths(case), _news(case)
    begin = np.concatenate([[0], np.cumsum(news)])
    table = st["table"].cpu().numpy()
    ks, vs = st["scales"]

    def cached(s, first, last, values=True):
        """Keys and values of one sequence's places first .. last - 1, [place, kv head, dim]."""
        ids = torch.from_numpy(table[s, first // page:(last - 1) // page + 1].astype(np.int64)).to(DEV)
        cut = slice(first - first // page * page, last - first // page * page)

        def line(pool):
            return pool[ids].transpose(1, 2).flatten(0, 1)[cut]

        if case["bits"] == 16:
            return line(st["k"]).double(), line(st["v"]).double()
        return _values64(line(st["k"]), line(ks)), _values64(line(st["v"]), line(vs))

    if case["op"] == "append":
        angle = torch.arange(st["max_len"], device=DEV)
        table64 = st["rope"].double()

        def turned(x, at):
            y = x.double().clone()
            for e in range(case["pairs"]):
                c, s = table64[at, e][:, None], table64[at, D // 2 + e][:, None]
                y[..., e] = x[..., e].double() * c - x[..., e + D // 2].double() * s
                y[..., e + D // 2] = x[..., e].double() * s + x[..., e + D // 2].double() * c
            return y

        q, kk, vv = [], [], []
        pk, pv = (st["k"].double(), st["v"].double()) if case["bits"] == 16 else (None, None)
        for s, (n, L) in enumerate(zip(news, lengths)):
            a, b = int(begin[s]), int(begin[s + 1])
            at = angle[L - n:L]
            q.append(turned(st["q"][a:b], at))
            k, v = turned(st["new_k"][a:b], at), st["new_v"][a:b].double()
            if case["bits"] == 16:
                ids = torch.from_numpy(table[s].astype(np.int64)).to(DEV)[at // page]
                for h in range(case["kv_heads"]):
                    pk[ids, h, at % page] = k[:, h]
                    pv[ids, h, at % page] = v[:, h]
            else:
                if L > n:
                    ck, cv = cached(s, 0, L - n)
                    kk.append(ck)
                    vv.append(cv)
                kk.append(_codes64(k))
                vv.append(_codes64(v))
        if case["bits"] == 16:
            return {"q": torch.cat(q), "k": pk, "v": pv}
        return {"q": torch.cat(q), "k": torch.cat(kk), "v": torch.cat(vv)}

    out = torch.zeros((st["tokens"], case["heads"], D), dtype=torch.float64, device=DEV)
    share = case["heads"] // case["kv_heads"]
    for s, (n, L) in enumerate(zip(news, lengths)):
        for a in range(0, n, 1024):  # queries in chunks, each over the keys that it can reach
            b = min(n, a + 1024)
            t = torch.arange(L - n + a, L - n + b, device=DEV)
            first = max(0, L - n + a + 1 - case["window"]) if case["window"] else 0
            places = [(0, min(case["sinks"], first))] if min(case["sinks"], first) else []
            places.append((first, L - n + b))
            got = [cached(s, *p) for p in places]
            k, v = torch.cat([g[0] for g in got]), torch.cat([g[1] for g in got])
            j = torch.cat([torch.arange(*p, device=DEV) for p in places])
            hidden = j[None] > t[:, None]
            if case["window"]:
                hidden |= (j[None] <= t[:, None] - case["window"]) & (j[None] >= case["sinks"])
            rows = slice(int(begin[s]) + a, int(begin[s]) + b)
            for h in range(case["heads"]):
                z = st["q"][rows, h].double() @ k[:, h // share].T * D ** -0.5
                z[hidden] = -math.inf
                out[rows, h] = torch.softmax(z, -1) @ v[:, h // share]
    return out
