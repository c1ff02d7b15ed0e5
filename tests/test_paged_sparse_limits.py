"""Decode over selected pages: sizes and numbers past what the kernels hold, refused before any launch and without a GPU."""

import math

import pytest
import torch

from hk_dsl_b200.ops import paged_sparse as ps
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


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-40, 2.0 ** 127, math.inf, math.nan])
def test_a_scale_that_fp32_does_not_hold_as_a_positive_number_is_refused(scale):
    bf = torch.bfloat16
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    cache, q = z(5, 16, 2, 64, dtype=bf), z(2, 8, 64, dtype=bf)
    with pytest.raises(ValueError, match="scale"):
        ps.paged_sparse_decode(torch.empty_like(q), q, cache, cache, z(2, 3), z(2), z(2, 2, 3), scale)
    with pytest.raises(ValueError, match="scale"):
        ps.page_scores(z(2, 2, 3, dtype=torch.float32), q, z(5, 2, 2, 64, dtype=bf), z(2, 3), z(2), scale, 16)
    l = lib.load()
    assert l.hkb_page_scores(lib.PAGE_SCORES(16, 16, 8, 8, 16, 512, 128, 16, 512, 256, 4, 16, 8, 16, 2, 4, 2, 128, 16, 0, 0, scale), None) == -10
    assert l.hkb_paged_sparse_decode(lib.SPARSE_DECODE(
        16, 512, 128, 0, 16, 512, 128, 16, 2048, 128, 32768, 4, 16, 2048, 128, 32768, 4, 16, 8, 8, 16, 16, 8, 4, 4, 2, 4, 2, 128, 16,
        0, 0, 0, scale), None) == -10
