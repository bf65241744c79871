"""The cache's C ABI at the edges of its arguments, without a GPU."""

import ctypes

import pytest
from test_kvcache_host import append, attention, cache, rows, step

from jitcast_b200 import _lib


@pytest.mark.parametrize("heads,tokens,ld,hs,good", [
    (4, 5, 64, 5 * 64, True),       # heads before tokens
    (4, 5, 64, 5 * 64 - 1, False),  # the next head's first row in this one's last
    (4, 5, 63, 5 * 64, False),      # rows of a head overlap
    (4, 5, 256, 64, True),
    (4, 5, 255, 64, False),
    (4, 5, 70, 4 * 70 + 64, True),  # with gaps
    (4, 5, 70, 4 * 70 + 63, False),
    (4, 1, 0, 64, True),            # one row has no pitch
    (1, 5, 64, 0, True),
    (1, 5, 63, 0, False),
    (4, 5, 1 << 40, 64, True),
    (4, 5, 64, (1 << 62), True),
])
def test_rows_that_a_call_writes(heads, tokens, ld, hs, good):
    # device 99 does not exist: what passes the checks ends there
    want = _lib.ERR_NO_DEVICE if good else _lib.ERR_INVALID_ARG
    s, c = step(tokens=tokens), cache(kv_heads=1)
    need = ctypes.c_longlong(-1)
    assert _lib.lib().jc_kv_attention_workspace(_lib.BF16, ctypes.byref(c), ctypes.byref(s), heads, 0, 0,
                                                ctypes.byref(need)) == _lib.OK
    assert attention(c=c, s=s, heads=heads, q=rows(hs=max(hs, 64)), out=rows(ld=ld, hs=hs), ws=64, ws_bytes=need.value) == want
    assert append(c=c, s=s, q=rows(), heads=heads, q_out=rows(ld=ld, hs=hs)) == want


def workspace(s, heads=2, kv_heads=2):
    need = ctypes.c_longlong(-1)
    c = cache(kv_heads=kv_heads, page_size=1 << 20, pages=1)
    st = _lib.lib().jc_kv_attention_workspace(_lib.BF16, ctypes.byref(c), ctypes.byref(s), heads, 0, 0, ctypes.byref(need))
    return st, need.value


@pytest.mark.parametrize("max_new", [6, 33, 1 << 20, (1 << 31) - 1])
def test_a_loose_bound_of_new_tokens_shapes_nothing(max_new):
    # at most 5 of 5 rows: one long sequence's keys are split as they are for the tight bound
    tight = workspace(step(tokens=5, max_new=5, max_length=100000))
    assert tight[0] == _lib.OK and tight[1] > 0
    assert workspace(step(tokens=5, max_new=max_new, max_length=100000)) == tight


def test_more_query_rows_than_a_launch_has():
    # (kv heads, heads, tokens): kernels and grids count rows of a sequence in 31 bits
    for kv, heads, tokens, good in ((64, 64, (1 << 24) + 1, False), (64, 64, 1 << 24, True), (1, 65535, 1 << 14, True),
                                    (1, 65535, (1 << 14) + 1, False)):
        for length in (1, 5000):
            st, _ = workspace(step(tokens=tokens, max_new=tokens, max_length=length), heads, kv)
            assert st == (_lib.OK if good else _lib.ERR_UNSUPPORTED_SHAPE), (kv, heads, tokens, length)
