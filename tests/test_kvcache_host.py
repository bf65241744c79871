"""The key/value cache's C ABI without a GPU: struct layouts, argument refusals before any device work, and the
workspace arithmetic."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from jitcast_b200 import _lib, kvcache

P = 64  # a pointer that is never followed


def cache(**kw):
    c = dict(bits=16, pages=8, page_size=32, kv_heads=2, head_dim=64, k=P, v=P, k_scale=None, v_scale=None)
    return kvcache._Cache(*{**c, **kw}.values())


def step(**kw):
    s = dict(sequences=2, tokens=5, max_new=3, max_length=90, start=P, length=P, page_table=P, table_pages=3, ld_table=3)
    return kvcache._Step(*{**s, **kw}.values())


def rows(data=P, ld=256, hs=64):
    return kvcache._Rows(data, ld, hs)


def attention(c=None, s=None, q=None, heads=4, out=None, window=0, sinks=0, scale=0.125, precision=_lib.BF16, ws=None,
              ws_bytes=0):
    r = ctypes.byref
    return _lib.lib().jc_kv_attention_device(99, precision, r(c or cache()), r(s or step()), r(q or rows()), heads,
                                             r(out or rows()), window, sinks, scale, ws, ws_bytes, None)


def append(c=None, s=None, k=None, v=None, q=None, heads=0, q_out=None, table=None, table_rows=0, pairs=0):
    r = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    return _lib.lib().jc_kv_append_device(99, _lib.FP16, r(c or cache()), r(s or step()), r(k or rows()), r(v or rows()),
                                          r(q), heads, r(q_out), None, table, table_rows, pairs, None)


@pytest.mark.parametrize("kw", [
    dict(bits=8), dict(pages=0), dict(kv_heads=0), dict(k=None), dict(v=None), dict(k=P + 2), dict(bits=4),
    dict(bits=4, k_scale=P), dict(bits=4, k_scale=P, v_scale=P + 4)])
def test_bad_caches(kw):
    assert attention(c=cache(**kw)) == _lib.ERR_INVALID_ARG
    assert append(c=cache(**kw)) == _lib.ERR_INVALID_ARG
    assert _lib.last_error()


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(page_size=40), dict(page_size=0), dict(head_dim=32),
                                dict(head_dim=96), dict(pages=1 << 30)])
def test_unsupported_caches(kw):
    assert attention(c=cache(**kw)) == _lib.ERR_UNSUPPORTED_SHAPE
    assert append(c=cache(**kw)) == _lib.ERR_UNSUPPORTED_SHAPE


@pytest.mark.parametrize("kw", [
    dict(sequences=-1), dict(tokens=-1), dict(max_new=-1), dict(max_length=-1), dict(table_pages=-1), dict(ld_table=2),
    dict(length=None), dict(page_table=None), dict(start=None), dict(start=None, tokens=2, max_new=2)])
def test_bad_steps(kw):
    assert attention(s=step(**kw)) == _lib.ERR_INVALID_ARG
    assert append(s=step(**kw)) == _lib.ERR_INVALID_ARG


def test_bad_attention_arguments():
    bad = [dict(heads=3), dict(heads=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("inf")), dict(scale=float("nan")), dict(precision=_lib.FP32), dict(precision=7),
           dict(q=rows(data=None)), dict(q=rows(data=P + 1)), dict(q=rows(hs=32)), dict(out=rows(ld=128)),
           dict(out=rows(hs=63)), dict(q=rows(ld=-1))]
    for kw in bad:
        assert attention(**kw) == _lib.ERR_INVALID_ARG, kw
    assert attention(s=step(sequences=70000)) == _lib.ERR_UNSUPPORTED_SHAPE


def test_bad_append_arguments():
    bad = [dict(k=rows(data=None)), dict(v=rows(data=P + 1)), dict(q=rows(), heads=0, q_out=rows()),
           dict(q=rows(), heads=4), dict(q=rows(), heads=4, q_out=rows(ld=64)), dict(table=P, table_rows=0, pairs=4),
           dict(table=P, table_rows=9, pairs=33), dict(table=P, table_rows=9, pairs=-1)]
    for kw in bad:
        assert append(**kw) == _lib.ERR_INVALID_ARG, kw


def test_good_arguments_reach_the_device_check():
    # device 99 does not exist: everything before it passed
    need = ctypes.c_longlong(-1)
    st = _lib.lib().jc_kv_attention_workspace(_lib.BF16, ctypes.byref(cache()), ctypes.byref(step()), 4, 0, 0,
                                              ctypes.byref(need))
    assert st == _lib.OK and need.value >= 0
    assert attention(ws=P, ws_bytes=need.value) == _lib.ERR_NO_DEVICE
    assert append(q=rows(), heads=4, q_out=rows(), table=P, table_rows=9, pairs=32) == _lib.ERR_NO_DEVICE
    r = ctypes.byref
    assert _lib.lib().jc_kv_read_device(99, _lib.BF16, r(cache()), r(step()), r(rows()), r(rows()), None) == \
        _lib.ERR_NO_DEVICE
    assert _lib.lib().jc_kv_attention_workspace(_lib.BF16, r(cache()), r(step()), 4, 0, 0, None) == _lib.ERR_INVALID_ARG


def test_struct_layouts_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    classes = {"jc_kv_cache": kvcache._Cache, "jc_kv_step": kvcache._Step, "jc_kv_rows": kvcache._Rows}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "jitcast_b200.h"', "int main(void) {"]
    want = []
    for c, cls in classes.items():
        lines.append(f'  printf("%zu\\n", sizeof({c}));')
        want.append(ctypes.sizeof(cls))
        for name, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({c}, {name}));')
            want.append(getattr(cls, name).offset)
    src, exe = tmp_path / "layouts.c", tmp_path / "layouts"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    inc = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-std=c11", "-I", str(inc), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == want


def test_rope_table_is_the_engines_rule():
    # cos and sin of FP32(position x FP32 frequency), frequencies theta^-(2e / 2 pairs); resting pairs 1 and 0
    t = kvcache.rope_table(40, 64, 16, 10000.0, device="cpu").numpy()
    freq = [np.float32(1) / np.float32(10000.0 ** float(np.float32(2 * e) / np.float32(32))) for e in range(16)]
    for p in (0, 1, 17, 39):
        for e in range(16):
            angle = float(np.float32(p) * freq[e])
            assert t[p, e] == np.float32(np.cos(angle)) and t[p, 32 + e] == np.float32(np.sin(angle))
    assert (t[:, 16:32] == 1).all() and (t[:, 48:] == 0).all()
