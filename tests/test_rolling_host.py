"""A rolling forecast's page bookkeeping, on the CPU."""

import pytest

from jitcast_b200.rolling import Pages

pytest.importorskip("torch")


def seen(length, window, sinks):
    """The indexes that the token at length - 1 sees."""
    return {j for j in range(length) if not window or j > length - 1 - window or j < sinks}


@pytest.mark.parametrize("page,window,sinks", [(32, 100, 3), (16, 16, 0), (16, 1, 0), (64, 40, 70), (16, 50, 16)])
def test_a_pool_of_the_windows_pages_is_enough(page, window, sinks):
    # several windows' worth of patches, one at a time: the pages that a step's tokens see, and no others for long
    most = 12 * window + 5 * page
    need = Pages.most(most, page, window, sinks)
    assert need <= -(-sinks // page) + (window + page - 2) // page + 1
    pages = Pages(2, 2 * need, page, most, device="cpu")
    held = [{}, {}]
    for length in range(1, most + 1):
        pages.grow([length, length])
        assert pages.used <= 2 * need
        for s in range(2):
            row = pages.table[s].tolist()
            for j in {j // page for j in seen(length, window, sinks)}:
                assert row[j] >= 0
                assert held[s].setdefault(j, row[j]) == row[j]  # a page that is seen stays where it is
        shown = [row[j // page] for row in pages.table.tolist() for j in seen(length, window, sinks)]
        assert len(set(shown)) == len({(s, j // page) for s in range(2) for j in seen(length, window, sinks)})
        pages.leave([length, length], window, sinks)
    assert pages.peak <= 2 * need


def test_pages_of_chunks_and_of_no_window():
    # a prompt, then chunks of 7: a pool of the most that such steps hold is enough; without a window all pages stay
    for window, sinks in ((90, 5), (0, 0)):
        need = Pages.most(700, 32, window, sinks, chunk=97)
        pages = Pages(1, need, 32, 700, device="cpu")
        for length in [97] + list(range(104, 701, 7)):
            pages.grow([length])
            pages.leave([length], window, sinks)
        assert pages.peak <= need
        if not window:
            assert need == pages.used == 22


def test_uneven_series_and_a_full_pool():
    pages = Pages(3, 6, 16, 200, device="cpu")
    pages.grow([40, 0, 17])
    assert pages.used == 5 and pages.table[1].tolist() == [-1] * 13
    with pytest.raises(RuntimeError):
        pages.grow([40, 40, 17])
    assert pages.used == 5  # nothing was taken by the call that failed
    pages.leave([40, 0, 17], 10, 0)  # the next tokens see 31 .. and 8 ..
    assert pages.used == 4
    pages.grow([48, 20, 17])
    assert pages.used == 6 and int((pages.table[1] >= 0).sum()) == 2


def test_what_a_step_reads_is_not_rewritten_under_it():
    # a copy that runs late, as one enqueued behind other work does: the table that it brings is the one of its grow
    class Late:
        def copy_(self, src, non_blocking=False):
            self.src = src

    pages = Pages(1, 9, 16, 300, device="cpu")
    pages.grow([90])
    first = pages.table.clone()
    pages.table = late = Late()
    pages.grow([110])
    pages.leave([110], 20, 0)  # most of the pages that the step just enqueued sees at its first tokens
    assert int((late.src[0] >= 0).sum()) == 7
    assert late.src[0, :6].tolist() == first[0, :6].tolist()
