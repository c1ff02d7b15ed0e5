"""Decode over selected pages where its contract is easily broken: refused requests, extreme and infinite values, wide
strides, the integers' ends, block tables past one chunk of requests, tables wider than every sequence."""

import math
import random

import pytest
import torch

from oracle import paged_oracle as dense
from oracle import sparse_oracle as orc
from test_gpu_paged_sparse import (BF, _Loop, _advance, _attend, _bounds_of, _cache_case, _check_attend, _cu, _hold,
                                   _lens, _ps, _random_pages, _same, _tables_case)

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


# ------------------------------------------------------------------------------ queries over an fp8 cache

@pytest.mark.parametrize("d, group, power", [(64, 4, 100), (128, 8, -100), (128, 12, 17), (256, 16, 100), (256, 3, -40)])
def test_fp8_attention_takes_queries_of_any_magnitude(d, group, power):
    """A power of two moved from the scale to the query changes no logit, and so no bit of the answer."""
    c = _cache_case([200, 1, 33], d=d, h_kv=2, group=group, kv="fp8", seed=d + group)
    pages = _random_pages(c, 6)
    want, lse = _attend(c, pages)
    _check_attend(c, pages, want, lse)
    c.update(q=(c["q"].float() * 2.0 ** power).to(BF), scale=c["scale"] * 2.0 ** -power)
    got, lse_p = _attend(c, pages)
    assert torch.equal(got, want) and torch.equal(lse_p, lse)


@pytest.mark.parametrize("d, group", [(64, 4), (128, 12), (256, 8)])
def test_fp8_attention_scales_every_head_by_itself(d, group):
    """Heads of one kv head between 2^-9 and 2^18, past fp16's 65504: logits up to some hundreds, as the oracle has them."""
    c = _cache_case([300, 17], d=d, h_kv=1, group=group, kv="fp8", seed=d)
    size = 2.0 ** torch.linspace(-9, 18, group)
    c.update(q=(c["q"].float() * size[None, :, None]).to(BF), scale=c["scale"] * 2.0 ** -10)
    assert float(c["q"].float().abs().max()) > 2 * 65504
    pages = _random_pages(c, 9)
    got, lse = _attend(c, pages)
    _check_attend(c, pages, got, lse)


@pytest.mark.parametrize("d, group", [(64, 4), (128, 12), (256, 8)])
def test_fp8_attention_shows_a_broken_query(d, group):
    """A NaN or infinite element makes its own head NaN (an infinite logit of either sign is among the keys') and no other."""
    c = _cache_case([300, 90, 40], d=d, h_kv=2, group=group, kv="fp8", seed=d)
    pages = _random_pages(c, 9)
    want, lse = _attend(c, pages)
    heads = c["q"].shape[1]
    bad = torch.zeros(3, heads, dtype=torch.bool)
    for r, (h, x) in enumerate([(1, math.nan), (heads - 1, math.inf), (group - 1, -math.inf)]):
        c["q"][r, h, 5 * r + 3] = x
        bad[r, h] = True
    got, lse_b = _attend(c, pages)
    assert torch.isnan(got[bad.cuda()]).all() and torch.isnan(lse_b[bad.cuda()]).all()
    assert torch.equal(got[~bad.cuda()], want[~bad.cuda()]) and torch.equal(lse_b[~bad.cuda()], lse[~bad.cuda()])


# ------------------------------------------------------------------------------ wide strides

def test_a_cache_whose_tokens_lie_hundreds_of_megabytes_apart():
    """Token-major across the whole pool, K and V side by side: seven tokens are more than 2^31 bytes."""
    from hk_dsl_b200.ops import paged
    nb, page, d = 2_400_000, 16, 64
    assert 7 * nb * 2 * d > 2 ** 31
    store = torch.empty(page, nb, 2, 1, d, dtype=torch.uint8, device="cuda")
    k8, v8 = store[:, :, 0].transpose(0, 1), store[:, :, 1].transpose(0, 1)
    ids = torch.tensor([[nb - 1, 0, nb // 2, nb - 2, 77], [5, nb // 3, 0, 0, 0]], dtype=torch.int32)
    lens, ks = [5 * page - 3, page + 1], torch.tensor([0.0125])
    g = torch.Generator().manual_seed(3)
    raw = dense.quantize_fp8(torch.randn(2, 10, page, 1, d, generator=g), ks)
    at = ids.flatten().unique()                # a page of its own for each id, the rest of the pool as it was
    k, v = raw[0, :at.numel()].view(torch.uint8), raw[1, :at.numel()].view(torch.uint8)
    for i, b in enumerate(at.tolist()):
        k8[b], v8[b] = k[i].cuda(), v[i].cuda()
    small = torch.searchsorted(at, ids).to(torch.int32)
    q = torch.randn(2, 8, d, generator=g).to(BF)
    pages = torch.tensor([[0, 2, 4], [0, 1, -1]], dtype=torch.int32).view(2, 1, 3)
    cu = lambda x: x.cuda()  # noqa: E731
    n = torch.tensor(lens, dtype=torch.int32).cuda()

    out, lse = torch.empty(2, 8, d, dtype=BF, device="cuda"), torch.empty(2, 8, device="cuda")
    _ps().paged_sparse_decode(out, cu(q), k8, v8, cu(ids), n, cu(pages), d ** -0.5, "fp8", cu(ks), cu(ks), out_lse=lse)
    want, tol, wl, tl = orc.sparse_ref(q, k, v, small, lens, pages, d ** -0.5, ks, ks)
    _hold(out, want, tol)
    _hold(lse, wl, tl)
    every = torch.arange(5, dtype=torch.int32).expand(2, 1, 5)
    paged.paged_attention_decode(out, cu(q), k8, v8, cu(ids), n, d ** -0.5, "fp8", cu(ks), cu(ks))
    want, tol, _, _ = orc.sparse_ref(q, k, v, small, lens, every, d ** -0.5, ks, ks)
    _hold(out, want, tol)
    bounds = torch.zeros(nb, 1, 2, d, dtype=torch.uint8, device="cuda")
    _ps().update_page_bounds(bounds, k8, cu(ids), n, cu(torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32)), num_tokens=sum(lens))
    want = orc.bounds_ref(torch.zeros(at.numel(), 1, 2, d, dtype=torch.uint8), k, small, lens, [0, lens[0], sum(lens)])
    assert _same(bounds[at.long().cuda()], want)


# ------------------------------------------------------------------------------ infinite summaries

@pytest.mark.parametrize("kv", ["bf16", "f16"])
@pytest.mark.parametrize("d, group", [(64, 1), (64, 4), (128, 8), (128, 12), (256, 5), (256, 16)])
def test_page_scores_of_infinite_bounds_are_the_definitions(kv, d, group):
    """max(q low, q high) is finite where the infinite bound is the lesser of the two products; a query of zero that meets an
    infinity is no number, and neither is a sum of both infinities."""
    c = _cache_case([16 * 39 + 5, 16 * 3], d=d, h_kv=2, group=group, kv=kv, seed=d + group)
    b = _bounds_of(c)
    g = torch.Generator().manual_seed(group)
    for p in range(39):                      # pages 20 to 23 and the last one keep finite bounds
        if p in (20, 21, 22, 23):
            continue
        for _ in range(1 + p % 3):
            h, x = int(torch.randint(2, (), generator=g)), int(torch.randint(d, (), generator=g))
            kind = p % 5
            low, high = b[int(c["table"][0, p]), h, :, x]
            b[int(c["table"][0, p]), h, :, x] = torch.tensor(
                [[float(low), math.inf], [-math.inf, float(high)], [-math.inf, math.inf], [math.inf, math.inf], [-math.inf, -math.inf]][kind])
    c["q"][0, 0, ::7] = 0.0
    c["q"][0, group, 1::7] = -0.0
    want, tol = orc.scores_ref(c["q"], b, c["table"], c["lens"], 16, c["scale"])
    fin = torch.isfinite(want[0, :, :39])
    assert 20 < int(fin.sum()) < 78 and torch.isfinite(tol[0, :, :39][fin]).all()
    got = torch.full(want.shape, 5.0, device="cuda")
    _ps().page_scores(got, c["q"].cuda(), b.cuda(), c["table"].cuda(), _lens(c), c["scale"], 16)
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isposinf(got), torch.isposinf(want))
    _hold(got, want, tol)


@pytest.mark.parametrize("kv", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("d, group", [(64, 4), (128, 12), (256, 16)])
def test_page_scores_of_a_broken_query(kv, d, group):
    """A NaN in any head of a group makes all pages of its row and kv head NaN, and no others."""
    c = _cache_case([16 * 30, 16 * 7 + 1, 400], d=d, h_kv=2, group=group, kv=kv, seed=d + group)
    b = _bounds_of(c)
    for r, h, x in ((0, 0, d - 1), (1, 2 * group - 1, 0), (2, group - 1, d // 2 + 1)):
        c["q"][r, h, x] = -math.nan if r else math.nan
    want, tol = orc.scores_ref(c["q"], b, c["table"], c["lens"], 16, c["scale"], c["ks"])
    assert torch.isnan(want[0, 0, :30]).all() and torch.isnan(want[1, 1, :8]).all() and torch.isfinite(want[0, 1, :30]).all()
    got = torch.full(want.shape, 5.0, device="cuda")
    _ps().page_scores(got, c["q"].cuda(), b.cuda(), c["table"].cuda(), _lens(c), c["scale"], 16, c["name"], _cu(c["ks"]))
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    _hold(got, want, tol)


# ------------------------------------------------------------------------------ the integers' ends

def test_advance_tables_takes_back_as_many_pages_as_an_int_counts():
    """One request gives back 2^31 - 1 pages of one token."""
    n = 2 ** 31 - 1
    table = torch.arange(n - 1, -1, -1, dtype=torch.int32, device="cuda").view(1, n)
    free = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, count, starts, status = i32(n), i32(0), i32(7, 7), i32(7)
    slots = torch.full((1,), 7, dtype=torch.int64, device="cuda")
    pos = slots.clone()
    _ps().advance_tables(table, lens, i32(-n), free, count, 1, slots, pos, starts, status)
    assert int(lens) == 0 and int(count) == n and int(status) == orc.OK and int(slots) == -1 and starts.tolist() == [0, 0]
    assert torch.equal(free, table[0])


def test_paged_sparse_decode_of_a_sequence_that_ends_where_ints_do():
    """The tile of positions 2^31 - 16 .. 2^31 - 1 holds 15 tokens of a sequence of 2^31 - 1; the last one is nobody's."""
    page, d, last = 16, 64, 2 ** 27 - 1
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(3, page, 1, d, generator=g).to(BF), torch.randn(3, page, 1, d, generator=g).to(BF)
    k[2, 15] = v[2, 15] = math.nan
    q = torch.randn(1, 4, d, generator=g).to(BF)
    table = torch.zeros(1, last + 1, dtype=torch.int32, device="cuda")
    table[0, last], table[0, last - 1] = 2, 1
    pages = torch.tensor([0, last - 1, last], dtype=torch.int32).view(1, 1, 3)
    out, lse = torch.empty(1, 4, d, dtype=BF, device="cuda"), torch.empty(1, 4, device="cuda")
    _ps().paged_sparse_decode(out, q.cuda(), k.cuda(), v.cuda(), table, torch.tensor([2 ** 31 - 1], dtype=torch.int32).cuda(),
                              pages.cuda(), d ** -0.5, out_lse=lse)
    want, tol, wl, tl = orc.sparse_ref(q, k, v, torch.tensor([[0, 1, 2]]), [47], torch.arange(3).view(1, 1, 3), d ** -0.5)
    _hold(out, want, tol)
    _hold(lse, wl, tl)


# ------------------------------------------------------------------------------ requests past one chunk of the scan

@pytest.mark.parametrize("n, page, width, pool, rows, first_short, first_cut", [
    (2049, 16, 4, 20000, 60000, None, None),       # a second chunk of one request
    (5000, 16, 6, 7700, 60000, 0, None),           # the free pages run out in the first chunk, and stay out
    (5000, 16, 6, 40000, 18000, None, 1),          # the rows in the second
    (6145, 5, 9, 13700, 15000, 1, 2),              # the pages in the second, the rows in the third
    (34821, 1, 3, 200000, 23000, None, 14),        # more chunks than the cluster has CTAs
])
def test_advance_tables_of_many_requests(n, page, width, pool, rows, first_short, first_cut):
    table, lens, new, free, count, rows = _tables_case(n, n, page, width, pool, rows)
    chunk = 2048
    for i in range(0, n, 1024):                    # somebody gives pages back in every chunk
        lens[i], new[i] = (0, 1) if lens[i] == 0 else (lens[i], -lens[i])
    want = orc.advance_ref(table, lens, new, free, count, page, rows)
    status = want[7]
    if first_short is not None:
        assert status.index(orc.NO_PAGES) // chunk == first_short
    if first_cut is not None:
        assert status.index(orc.NO_ROWS) // chunk == first_cut
    assert all(any(m < 0 < k for m, k in zip(new[c:c + chunk], lens[c:c + chunk])) for c in range(0, n - 1, chunk))
    got = _advance(table, lens, new, free, count, page, rows)
    for name, g, w in zip(("table", "lens", "free", "count", "slots", "positions", "starts", "status"), got, want):
        assert g == w, name


# ------------------------------------------------------------------------------ wide tables, rows of one sequence

@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("width", [300, 700, 3000, 17000])
def test_a_table_far_wider_than_its_sequences(kv, width):
    """As a captured step has it: scores, selection and attention answer as with a table that just holds them, whatever the
    spare columns hold."""
    c = _cache_case([16 * 40, 1, 0, 16 * 9 + 5], d=128, h_kv=2, group=4, kv=kv, seed=width)
    b, tight = _bounds_of(c), c["table"].shape[1]
    q, ks, lens = c["q"].cuda(), _cu(c["ks"]), _lens(c)
    table = torch.full((4, width), 2 ** 31 - 1, dtype=torch.int32)
    table[:, :tight] = c["table"]
    answers = []
    for t in (c["table"], table):
        scores = torch.full((4, 2, t.shape[1]), 9.0, device="cuda")
        _ps().page_scores(scores, q, b.cuda(), t.cuda(), lens, c["scale"], 16, c["name"], ks)
        pages = torch.full((4, 2, 12), 99, dtype=torch.int32, device="cuda")
        _ps().select_pages(pages, scores, lens, 16, first=1, last=2)
        out, lse = _attend(c, pages.cpu(), table=t)
        answers.append((scores, pages, out, lse))
    (s0, p0, o0, l0), (s1, p1, o1, l1) = answers
    assert torch.equal(s1[:, :, :tight], s0) and torch.isneginf(s1[:, :, tight:]).all()
    assert torch.equal(p0.cpu(), orc.select_ref(s0.cpu(), c["lens"], 16, 12, 1, 2))
    assert torch.equal(p1, p0) and torch.equal(o1, o0) and torch.equal(l1, l0)
    _check_attend(c, p0.cpu(), o0, l0)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_several_tokens_of_one_sequence(kv):
    """Drafts: a query row for each of a sequence's last tokens, its table row repeated (by `expand` too), one length each."""
    c = _cache_case([333, 64], d=64, h_kv=2, group=4, kv=kv, seed=7)
    b = _bounds_of(c)
    rows = [(0, 330), (0, 331), (0, 332), (0, 333), (1, 63), (1, 64)]
    lens = [n for _, n in rows]
    table = c["table"][[r for r, _ in rows]].contiguous()
    g = torch.Generator().manual_seed(8)
    c.update(table=table, lens=lens, q=torch.randn(6, 8, 64, generator=g).to(BF))
    want, tol = orc.scores_ref(c["q"], b, table, lens, 16, c["scale"], c["ks"])
    scores = torch.zeros(want.shape, device="cuda")
    _ps().page_scores(scores, c["q"].cuda(), b.cuda(), table.cuda(), _lens(c), c["scale"], 16, c["name"], _cu(c["ks"]))
    _hold(scores, want, tol)
    pages = torch.zeros(6, 2, 9, dtype=torch.int32, device="cuda")
    _ps().select_pages(pages, scores, _lens(c), 16, first=1, last=2)
    assert torch.equal(pages.cpu(), orc.select_ref(scores.cpu(), lens, 16, 9, 1, 2))
    out, lse = _attend(c, pages.cpu())
    _check_attend(c, pages.cpu(), out, lse)
    part = dict(c, table=table[:1].cuda().expand(4, -1), lens=lens[:4], q=c["q"][:4])      # a row stride of 0
    got, _ = _attend(part, pages[:4].cpu())
    assert torch.equal(got, out[:4])


# ------------------------------------------------------------------------------ weights

@pytest.mark.parametrize("d, group, budget", [(64, 4, 12), (128, 8, 30), (256, 12, 7)])
def test_bf16_weights_are_not_rounded_to_bf16(d, group, budget):
    """Logits of nearly nothing, so that the weights' own rounding would be seen: they are held to 2^-15, not bf16's 2^-8."""
    c = _cache_case([200, 37, 480], d=d, h_kv=2, group=group, seed=d + 1)
    c["scale"] = 2.0 ** -12
    pages = _random_pages(c, budget)
    got, lse = _attend(c, pages)
    want, tol, wl, tl = orc.sparse_ref(c["q"], c["k"], c["v"], c["table"], c["lens"], pages, c["scale"], terms=2)
    _hold(got, want, tol)
    _hold(lse, wl, tl)


@pytest.mark.parametrize("kv", ["bf16", "f16"])
def test_an_infinite_value_makes_its_channel_infinite(kv):
    """Its weight is positive; no other channel, head or row changes, and behind a sequence's end it is not met."""
    c = _cache_case([300, 90, 37], d=128, h_kv=2, group=4, kv=kv, seed=19)
    pages = _random_pages(c, 20)
    want, lse = _attend(c, pages)
    c["v"][int(c["table"][0, 3]), 5, 1, 77] = math.inf
    c["v"][int(c["table"][1, 5]), 9, 0, 3] = -math.inf
    c["v"][int(c["table"][2, 2]), 5, 0, 9] = math.inf         # position 37 of 37 tokens
    got, lse2 = _attend(c, pages)
    hit = torch.zeros(want.shape, dtype=torch.bool)
    hit[0, 4:, 77] = hit[1, :4, 3] = True
    assert torch.isposinf(got[0, 4:, 77]).all() and torch.isneginf(got[1, :4, 3]).all()
    assert torch.equal(got[~hit.cuda()], want[~hit.cuda()]) and torch.equal(lse2, lse)
