"""The rolling forecast's layers (append, attention over the cache, page recycling) fed patch by patch against the same
layers fed all at once. Both round q, k, v, the probabilities and the attention's output to FP16 (2^-12 of a value on
average, each) and the projections' operands; two layers of a few such roundings each stay well below 1e-2 of the
output's norm. A 4-bit cache holds the same codes either way, up to a value whose FP16 inputs differ: bar 2e-2."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,bar", [(16, 1e-2), (4, 2e-2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_patch_by_patch_matches_all_at_once(jc, bits, bar, window, sinks, dim):
    pytest.importorskip("torch")
    from jitcast_b200 import ops, rolling

    rolled, whole, used = rolling.demo(series=5, patches=210, prompt=97, heads=2, dim=dim, bits=bits, window=window,
                                       sinks=sinks, page_size=32)
    ops.device_sync()
    err = float((rolled - whole).norm() / whole.norm())
    print(f"bits {bits} window {window}: {err:.2e}, {used} pages")
    assert err < bar
    if window:  # 210 patches are 7 pages a series; a window of 100 and a page of sinks keep at most 1 + 5
        assert used <= 5 * 6
    else:
        assert used == 5 * 7
