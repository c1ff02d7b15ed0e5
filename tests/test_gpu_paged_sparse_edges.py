"""Decode over selected pages where its contract is easily broken: refused requests, extreme and infinite values, wide
strides, the integers' ends, block tables past one chunk of requests, tables wider than every sequence."""

import random

import pytest
import torch

from oracle import sparse_oracle as orc
from test_gpu_paged_sparse import _Loop, _cache_case, _cu, _lens, _ps, _same

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------ summaries behind a refusal

@pytest.mark.parametrize("refused, behind", [([120, 100, 1, 1, -2], 4), ([200, 0, 0, -3, 0], 3), ([161, 2 ** 30, -5, 1, -12], 4)])
def test_a_step_summarises_shortened_pages_behind_a_request_refused_for_rows(refused, behind):
    """`query_start_loc` runs on past the step's rows where a request got none; the sequences behind it are summarised
    all the same."""
    s = _Loop(5)
    model = [[] for _ in range(5)]
    for i, new in enumerate(([40, 30, 20, 13, 33], refused)):
        s.fill(i, new)
        s.step()
        s.follow(model, new)
        if i == 0:
            s.check(model)
    assert orc.NO_ROWS in s.status.tolist() and s.status.tolist()[behind] == orc.OK and int(s.starts[5]) > s.rows
    s.check(model)


@pytest.mark.parametrize("page", [1, 16, 48])
@pytest.mark.parametrize("rows", [0, 1, 16, 77])
def test_page_bounds_of_starts_past_the_steps_rows(page, rows):
    """Tokens at or past row `num_tokens` are none: a sequence whose rows lie there has its last page summarised."""
    rnd = random.Random(page + rows)
    n = 300
    lens = [rnd.randint(0, 3 * page + 2) for _ in range(n)]
    starts = [0]
    for m in lens:
        starts.append(min(starts[-1] + rnd.choice([0, 1, min(m, 3), m, 10 ** 9]), 2 ** 31 - 1))
    c = _cache_case(lens, d=64, h_kv=1, page=page, seed=rows)
    b0 = _ps().page_bounds(c["k"]).copy_(torch.ones(()))
    b = _cu(b0)
    _ps().update_page_bounds(b, _cu(c["k"]), _cu(c["table"]), _lens(c), torch.tensor(starts, dtype=torch.int32).cuda(),
                             num_tokens=rows)
    assert _same(b, orc.bounds_ref(b0, c["k"], c["table"], lens, [min(s, rows) for s in starts]))
