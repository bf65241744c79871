"""The rolling forecast on a pool that holds what its window needs, over several windows' worth of patches, against the same
layers fed all at once on a pool for everything. The bars are those of test_rolling_gpu.py."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,bar", [(16, 1e-2), (4, 2e-2)])
def test_a_windows_pool_over_many_windows(jc, bits, bar):
    pytest.importorskip("torch")
    from jitcast_b200 import ops, rolling

    rolled, whole, used = rolling.demo(series=3, patches=700, prompt=60, heads=2, dim=64, bits=bits, window=100, sinks=3,
                                       page_size=32)
    ops.device_sync()
    assert used <= 3 * (1 + 5)  # of 22 pages a series
    assert float((rolled - whole).norm() / whole.norm()) < bar


def test_pages_may_run_ahead_of_the_gpu(jc):
    # tables and frees enqueued behind other work: each step reads the table of its own grow
    torch = pytest.importorskip("torch")
    from jitcast_b200 import rolling

    pages = rolling.Pages(2, 40, 16, 4000)
    got, want = [], []
    torch.cuda._sleep(200_000_000)  # some 0.1 s of work before the first copy
    for length in range(90, 1500, 10):
        pages.grow([length, length])
        got.append(pages.table.clone())
        want.append(pages.host.copy())
        pages.leave([length, length], 40, 16)
    torch.cuda.synchronize()
    assert all((g.cpu().numpy()[w >= 0] == w[w >= 0]).all() for g, w in zip(got, want))


def test_projections_past_fp16_saturate(jc):
    # keys of 1e5 are held as 65504, as the engines hold them: an infinity that rotates by a sine of 0 is undefined
    torch = pytest.importorskip("torch")
    from jitcast_b200 import kvcache, ops, rolling

    w_qkv = torch.zeros((3 * 64, 64), device="cuda")
    w_qkv[64, 0] = 1e5 / 8
    w_qkv[128:, 0] = 1.0 / 8
    layer = rolling.RollingTimeAttention(w_qkv, torch.eye(64, device="cuda"), 1, 1, rope=kvcache.rope_table(4, 64))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    x = torch.zeros((1, 64), device="cuda")
    x[0, 0] = 8.0
    y = layer(x, kvcache.Step(i32([1]), i32([[0]]), 1))
    ops.device_sync()
    assert float(layer.cache.k[0, 0, 0, 0]) == 65504.0
    assert torch.equal(y - x, torch.ones_like(x))
