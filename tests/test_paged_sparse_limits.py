"""Decode over selected pages: sizes that the kernels' counters do not reach, refused before any launch and without a GPU."""

from hk_dsl_b200.runtime import lib


def test_sizes_past_the_kernels_counters_are_refused():
    """A counter that runs up to a size in steps must not pass 2^31: columns, budgets and summarised pages end at 2^30."""
    l, most = lib.load(), 2 ** 30

    def sel(budget, cols):
        return l.hkb_select_pages(lib.SELECT_PAGES(16, budget, budget, budget, 16, cols, cols, cols, 16, 1, 1, 16, 1, 4), None)

    def sco(cols):
        return l.hkb_page_scores(lib.PAGE_SCORES(16, cols, cols, cols, 16, 512, 128, 16, 512, 256, 4, 16, cols, 16, 1, 4, 2, 128,
                                                 16, 0, 0, 0.1), None)

    def bnd(page):
        return l.hkb_page_bounds(lib.PAGE_BOUNDS(16, 256, 256, 4, 16, 2048, 128, 32768, 4, 16, 4, 4, 16, 0, 1, 4, 1, 128, page, 0), None)

    for past in (most + 1, 2 ** 31 - 16384, 2 ** 31 - 1):
        assert sel(8, past) == sel(past, 20) == sco(past) == -9 and bnd(past) == -3
