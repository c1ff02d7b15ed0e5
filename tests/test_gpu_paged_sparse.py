"""Decode over selected pages and the page bookkeeping under it, against the float64 oracle.

Whole numbers are held to be equal; floating values to the bounds that the oracle counts from each kernel's roundings
(`oracle/sparse_oracle.py`). Sizes go where the kernels can go wrong: lengths of zero and one, pages that end inside a
tile, pages larger than a tile, groups that fill no column tile, strides, poisoned memory behind a sequence."""

import math
import random

import pytest
import torch

from oracle import paged_oracle as dense
from oracle import sparse_oracle as orc

pytestmark = pytest.mark.gpu

BF, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _ps():
    from hk_dsl_b200.ops import paged_sparse
    return paged_sparse


# ------------------------------------------------------------------------------ tables

def _tables_case(seed, n, page, width, pool, rows, steps=None):
    rnd = random.Random(seed)
    lens = [rnd.choice([0, 1, rnd.randint(0, page * width)]) for _ in range(n)]
    perm = rnd.sample(range(pool), pool)
    table = [[-7] * width for _ in range(n)]
    for i in range(n):
        k = orc.ceil_div(lens[i], page)
        if k > len(perm):
            lens[i], k = 0, 0
        for j in range(k):
            table[i][j] = perm.pop()
    free = perm + [-9] * (pool - len(perm))
    new = [rnd.choice([0, 1, 1, 1, 2, rnd.randint(1, page * width), -1, -rnd.randint(1, page * width), -(2 ** 31)])
           for _ in range(n)]
    return table, lens, new, free, len(perm), rows


def _advance(table, lens, new, free, count, page, rows, spare_cols=0):
    ps = _ps()
    width = len(table[0])
    store = torch.full((len(lens), width + spare_cols), 12345, dtype=torch.int32)
    store[:, :width] = torch.tensor(table, dtype=torch.int32)
    store = store.cuda()
    t = store[:, :width]
    cu = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    ln, fr, ct = cu(lens), cu(free), cu([count])
    slots = torch.full((rows,), 77, dtype=torch.int64, device="cuda")
    pos = torch.full((rows,), 77, dtype=torch.int64, device="cuda")
    starts, status = cu([55] * (len(lens) + 1)), cu([55] * len(lens))
    ps.advance_tables(t, ln, cu(new), fr, ct, page, slots, pos, starts, status)
    torch.cuda.synchronize()
    if spare_cols:
        assert (store[:, width:] == 12345).all()
    return (t.tolist(), ln.tolist(), fr.tolist(), int(ct), slots.tolist(), pos.tolist(), starts.tolist(), status.tolist())


@pytest.mark.parametrize("n, page, width, pool, rows, spare", [
    (1, 16, 3, 5, 40, 0), (7, 16, 6, 40, 200, 3), (64, 16, 20, 900, 2000, 0), (64, 5, 9, 200, 500, 0),
    (200, 1, 7, 1000, 900, 1), (513, 16, 8, 3000, 9001, 0), (1100, 48, 5, 4000, 60000, 0), (3, 64, 2, 0, 10, 0),
    (33, 16, 40, 4000, 0, 0),
])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_advance_tables(n, page, width, pool, rows, spare, seed):
    table, lens, new, free, count, rows = _tables_case(seed, n, page, width, pool, rows)
    want = orc.advance_ref(table, lens, new, free, count, page, rows)
    got = _advance(table, lens, new, free, count, page, rows, spare)
    for name, g, w in zip(("table", "lens", "free", "count", "slots", "positions", "starts", "status"), got, want):
        assert g == w, name


def test_advance_tables_many_steps_keep_every_page():
    """Steps after steps on the device alone: no page is lost or owned twice, and the oracle agrees at every step."""
    page, width, pool, n, rows = 16, 12, 90, 12, 128
    rnd = random.Random(5)
    table, lens = [[0] * width for _ in range(n)], [0] * n
    free, count = rnd.sample(range(pool), pool), pool
    for _ in range(25):
        new = [rnd.choice([0, 1, 1, 40, -1, -7, -1000]) for _ in range(n)]
        want = orc.advance_ref(table, lens, new, free, count, page, rows)
        got = _advance(table, lens, new, free, count, page, rows)
        assert list(got) == list(want)
        table, lens, free, count = got[:4]
        owned = [p for r, m in zip(table, lens) for p in r[:orc.ceil_div(m, page)]]
        assert sorted(owned + free[:count]) == list(range(pool))


def test_advance_tables_at_the_ends_of_its_integers():
    """Lengths and demands near 2^31, and a demand that goes past it."""
    top = 2 ** 31 - 1
    for page, width in ((1, 3), (16, 3), (2 ** 30, 2), (top, 1)):
        lens = [top, 5, 0, -3, 7, 2, top]
        new = [top, top, -top - 1, 1, top - 7, 0, -top]
        table = [[40 + i] * width for i in range(7)]
        want = orc.advance_ref(table, lens, new, [9, 8, 7, 6], 4, page, 4)
        got = _advance(table, lens, new, [9, 8, 7, 6], 4, page, 4)
        starts = [min(x, top) for x in want[6]]       # held at 2^31 - 1
        for name, g, w in zip(("table", "lens", "free", "count", "slots", "positions", "starts", "status"), got, want[:6] + (starts, want[7])):
            assert g == w, (page, name)


def test_advance_tables_without_requests_and_past_the_stacks_capacity():
    ps = _ps()
    e = lambda *s, d=torch.int32: torch.full(s, 9, dtype=d, device="cuda")  # noqa: E731
    slots, pos, starts, count = e(5, d=torch.int64), e(5, d=torch.int64), e(1), e(1)
    ps.advance_tables(e(0, 4), e(0), e(0), e(9), count, 16, slots, pos, starts, e(0))
    assert slots.tolist() == [-1] * 5 and pos.tolist() == [0] * 5 and starts.tolist() == [0] and int(count) == 9
    # a stack of two entries that three pages come back to: two stay, nothing is written behind them
    got = _advance([[4, 5, 6]], [48], [-48], [0, 0], 0, 16, 3)
    assert got[1] == [0] and got[2] == [4, 5] and got[3] == 2


# ------------------------------------------------------------------------------ caches

def _cache_case(lens, *, d=64, h_kv=2, group=4, page=16, kv="bf16", seed=0, layout="hnd", nan_tail=True, spare=3):
    g = torch.Generator().manual_seed(seed)
    act = F16 if kv == "f16" else BF
    pages = [max(1, orc.ceil_div(max(0, n), page)) for n in lens]
    nb, width = sum(pages) + spare, max(pages) + 1
    shape = (nb, h_kv, page, d) if layout == "hnd" else (nb, page, h_kv, d)
    k, v = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
    if layout == "hnd":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    ks = vs = None
    if kv == "fp8":
        ks, vs = torch.tensor([0.0125]), torch.tensor([0.011])
        k, v = dense.quantize_fp8(k, ks), dense.quantize_fp8(v, vs)
    else:
        k, v = k.to(act), v.to(act)
    perm = torch.randperm(nb, generator=g)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = perm[at:at + n].to(torch.int32)
        at += n
    if nan_tail:       # every token that no sequence holds
        live = torch.zeros(nb, page, dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(orc.ceil_div(max(0, n), page)):
                live[int(table[i, j]), :min(page, n - j * page)] = True
        dead = ~live[:, :, None, None].expand(k.shape)
        for c in (k, v):
            if kv == "fp8":
                c.view(torch.uint8)[dead] = 0x7f
            else:
                c[dead] = float("nan")
    q = torch.randn(len(lens), h_kv * group, d, generator=g).to(act)
    return dict(k=k, v=v, table=table, lens=list(lens), q=q, ks=ks, vs=vs, page=page, kv=kv, h_kv=h_kv,
                scale=d ** -0.5, name="fp8" if kv == "fp8" else "auto")


def _cu(t):
    return t.cuda() if isinstance(t, torch.Tensor) else t


def _lens(c):
    return torch.tensor(c["lens"], dtype=torch.int32).cuda()


def _same(a, b):
    """Bit for bit but for the sign of zero and a NaN's payload."""
    f = lambda x: (x.view(F8) if x.dtype == torch.uint8 else x).float().cpu()  # noqa: E731
    return torch.equal(torch.nan_to_num(f(a), nan=1e30), torch.nan_to_num(f(b), nan=1e30))


@pytest.mark.parametrize("kv", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("d, page, layout", [(64, 16, "hnd"), (128, 16, "nhd"), (128, 48, "hnd"), (256, 32, "nhd"), (64, 5, "nhd"),
                                             (128, 272, "hnd")])
def test_page_bounds_of_the_newest_tokens(kv, d, page, layout):
    lens = [1, page - 1, page, page + 1, 3 * page + 2, 0, 2 * page]
    c = _cache_case(lens, d=d, page=page, kv=kv, layout=layout, seed=page)
    b0 = _ps().page_bounds(c["k"]).copy_(torch.zeros(()))
    b = _cu(b0)
    _ps().update_page_bounds(b, _cu(c["k"]), _cu(c["table"]), _lens(c))
    assert _same(b, orc.bounds_ref(b0, c["k"], c["table"], lens))


@pytest.mark.parametrize("kv, page", [("bf16", 16), ("fp8", 16), ("f16", 48), ("bf16", 1)])
@pytest.mark.parametrize("n", [1, 5, 70, 1100])
def test_page_bounds_of_a_ragged_step(kv, page, n):
    rnd = random.Random(n + page)
    lens = [rnd.choice([0, 1, page, rnd.randint(1, 5 * page + 3)]) for _ in range(n)]
    new = [rnd.choice([0, min(m, 1), rnd.randint(0, m), m]) for m in lens]
    starts = [0]
    for k in new:
        starts.append(starts[-1] + k)
    c = _cache_case(lens, d=64, h_kv=3, page=page, kv=kv, seed=n)
    b0 = _ps().page_bounds(c["k"]).copy_(torch.ones(()))
    b = _cu(b0)
    _ps().update_page_bounds(b, _cu(c["k"]), _cu(c["table"]), _lens(c), torch.tensor(starts, dtype=torch.int32).cuda(),
                             num_tokens=starts[-1] + 9)
    assert _same(b, orc.bounds_ref(b0, c["k"], c["table"], lens, starts))


def test_page_bounds_keep_nan_and_infinity_and_skip_bad_pages():
    c = _cache_case([40, 33], d=64, seed=3)
    k = c["k"]
    k[int(c["table"][0, 2]), 3, 0, 5] = float("nan")
    k[int(c["table"][0, 2]), 4, 1, 6] = float("inf")
    k[int(c["table"][1, 2]), 0, 0, 7] = float("-inf")
    c["table"][1, 1] = 10 ** 6           # not a page of the pool
    b0 = torch.zeros_like(_ps().page_bounds(k))
    b = b0.cuda()
    starts = torch.tensor([0, 30, 50], dtype=torch.int32)
    _ps().update_page_bounds(b, k.cuda(), c["table"].cuda(), _lens(c), starts.cuda(), num_tokens=50)
    want = orc.bounds_ref(b0, k, c["table"], c["lens"], starts.tolist())
    assert torch.isnan(want[int(c["table"][0, 2]), 0, :, 5]).all() and _same(b, want)
    raw = k.float().clamp(-400, 400).nan_to_num(1.0).to(F8)         # uint8 storage is e4m3's bytes
    b8 = torch.zeros(b0.shape, dtype=torch.uint8, device="cuda")
    _ps().update_page_bounds(b8, raw.view(torch.uint8).cuda(), c["table"].cuda(), _lens(c))
    assert _same(b8, orc.bounds_ref(torch.zeros(b0.shape, dtype=torch.uint8), raw.view(torch.uint8), c["table"], c["lens"]))


# ------------------------------------------------------------------------------ scores

def _bounds_of(c):
    """A summary of every page of the case, live tokens only."""
    b = torch.zeros_like(_ps().page_bounds(c["k"]).view(torch.uint8) if c["kv"] == "fp8" else _ps().page_bounds(c["k"]))
    b = b.view(F8) if c["kv"] == "fp8" else b
    starts = [0]
    for n in c["lens"]:
        starts.append(starts[-1] + max(0, n))
    return orc.bounds_ref(b, c["k"], c["table"], c["lens"], starts)


def _hold(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(torch.isneginf(got), torch.isneginf(want)), what
    fin = torch.isfinite(want)
    assert torch.isfinite(got[fin]).all(), what
    off = (got[fin] - want[fin]).abs()
    assert (off <= tol[fin]).all(), f"{what}: {float((off / tol[fin].clamp_min(1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("kv", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("d, h_kv, group, page", [(64, 2, 4, 16), (128, 8, 4, 16), (128, 1, 16, 32), (256, 2, 7, 16), (64, 1, 1, 48),
                                                  (256, 1, 12, 16), (128, 3, 8, 5)])
def test_page_scores(kv, d, h_kv, group, page):
    lens = [1, 0, page, 7 * page + 3, 40 * page + 1, 16 * page, 17 * page]
    c = _cache_case(lens, d=d, h_kv=h_kv, group=group, page=page, kv=kv, seed=d + group)
    b = _bounds_of(c)
    want, tol = orc.scores_ref(c["q"], b, c["table"], lens, page, c["scale"], c["ks"])
    got = torch.full(want.shape, 5.0, device="cuda")
    _ps().page_scores(got, c["q"].cuda(), b.cuda(), c["table"].cuda(), _lens(c), c["scale"], page, c["name"], _cu(c["ks"]))
    _hold(got, want, tol)


def test_page_scores_strides_many_pages_and_extreme_queries():
    c = _cache_case([9000, 20], d=64, h_kv=2, group=3, kv="fp8", seed=2)
    b = _bounds_of(c)
    c["q"][0] *= 2.0 ** 100              # bf16 reaches far past fp16: the kernel scales by powers of two
    c["q"][1] *= 2.0 ** -100
    want, tol = orc.scores_ref(c["q"], b, c["table"], c["lens"], 16, c["scale"], c["ks"])
    q = torch.zeros(2, 6, 3 * 64, dtype=BF, device="cuda")[:, :, 64:128]
    q.copy_(c["q"])
    store = torch.zeros(b.shape[0], 2, 3, 64, device="cuda").to(F8)
    bb = store[:, :, :2]
    bb.copy_(b)
    got = torch.full((2, 2, want.shape[2] + 7), 5.0, device="cuda")[:, :, :want.shape[2]]
    _ps().page_scores(got, q, bb, c["table"].cuda(), _lens(c), c["scale"], 16, "fp8", c["ks"].cuda())
    _hold(got, want, tol)


def test_page_scores_nan_and_infinite_summaries():
    """A NaN or infinite bound shows in its own page's score and in no other."""
    c = _cache_case([16 * 20], d=64, h_kv=1, group=4, seed=4)
    b = _bounds_of(c)
    b[int(c["table"][0, 3]), 0, 1, 9] = float("nan")
    b[int(c["table"][0, 18]), 0, 1, 9] = float("inf")
    c["q"][0, :, 9] = 0.5
    want, tol = orc.scores_ref(c["q"], b, c["table"], c["lens"], 16, c["scale"])
    got = torch.zeros(want.shape, device="cuda")
    _ps().page_scores(got, c["q"].cuda(), b.cuda(), c["table"].cuda(), _lens(c), c["scale"], 16)
    got = got.cpu()
    assert math.isnan(got[0, 0, 3]) and got[0, 0, 18] == math.inf
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[0, 0, 3] = keep[0, 0, 18] = False
    _hold(got[keep], want[keep], tol[keep])


# ------------------------------------------------------------------------------ selection

def _select(x, lens, page, budget, first, last):
    out = torch.full((x.shape[0], x.shape[1], budget), 99, dtype=torch.int32, device="cuda")
    _ps().select_pages(out, x.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), page, first=first, last=last)
    return out.cpu()


@pytest.mark.parametrize("width", [1, 31, 64, 257, 1000, 2000, 2049, 4097, 9000, 16385, 40000])
@pytest.mark.parametrize("budget, first, last", [(1, 0, 0), (1, 1, 0), (5, 1, 4), (64, 1, 4), (300, 2, 0), (700, 0, 3)])
def test_select_pages(width, budget, first, last):
    g = torch.Generator().manual_seed(width)
    page = 16
    lens = [width * page, max(1, width * page // 2), 1, 0, width * page - 7, width * page + 1000]
    for name, x in (("normal", torch.randn(6, 2, width, generator=g)), ("ties", torch.randint(-2, 3, (6, 2, width), generator=g).float()),
                    ("one value", torch.full((6, 2, width), -3.5)), ("close", 18 + torch.randn(6, 2, width, generator=g) * 1e-5)):
        got = _select(x, lens, page, budget, first, last)
        assert torch.equal(got, orc.select_ref(x, lens, page, budget, first, last)), name


def test_select_pages_special_values():
    x = torch.randn(1, 1, 300, generator=torch.Generator().manual_seed(0))
    x[0, 0, 40], x[0, 0, 77], x[0, 0, 200], x[0, 0, 201] = math.nan, -math.nan, math.inf, -math.inf
    x[0, 0, 100:140:2], x[0, 0, 101:140:2] = 0.0, -0.0          # one value: ties in page order
    for budget in (2, 3, 4, 10, 120, 150, 299):
        assert torch.equal(_select(x, [300 * 16], 16, budget, 0, 1), orc.select_ref(x, [300 * 16], 16, budget, 0, 1)), budget
    x[:] = -math.inf
    assert _select(x, [300 * 16], 16, 6, 1, 2)[0, 0].tolist() == [0, 1, 2, 3, 298, 299]
    x[:] = math.nan
    assert _select(x, [300 * 16], 16, 6, 1, 2)[0, 0].tolist() == [0, 1, 2, 3, 298, 299]


def test_select_pages_reads_no_column_behind_the_sequence_and_takes_strides():
    x = torch.randn(3, 2, 50, generator=torch.Generator().manual_seed(1))
    want = orc.select_ref(x, [16 * 30] * 3, 16, 7, 1, 1)
    big = torch.full((3, 2, 90), math.inf, device="cuda")
    big[:, :, :30] = x[:, :, :30].cuda()
    store = torch.full((3, 2, 11), 5, dtype=torch.int32, device="cuda")
    _ps().select_pages(store[:, :, :7], big[:, :, :50], torch.full((3,), 16 * 30, dtype=torch.int32).cuda(), 16, first=1, last=1)
    assert torch.equal(store[:, :, :7].cpu(), want) and (store[:, :, 7:] == 5).all()


def test_select_pages_of_scores_that_share_a_histogram_bin():
    """Keys in three far groups, the border inside one of them: every level of the digits is gone through."""
    for width in (3000, 20000):
        x = torch.empty(1, 1, width)
        g = torch.Generator().manual_seed(width)
        x[0, 0] = torch.where(torch.rand(width, generator=g) < 0.3, -1e30, 1.0)
        near = torch.randint(0, 4, (width,), generator=g).float() * 2.0 ** -23 + 2.0
        x[0, 0] = torch.where(torch.rand(width, generator=g) < 0.5, near, x[0, 0])
        for budget in (1, 100, width // 4, width // 2, width - 1):
            assert torch.equal(_select(x, [width * 16], 16, budget, 0, 0), orc.select_ref(x, [width * 16], 16, budget, 0, 0)), budget


# ------------------------------------------------------------------------------ attention

def _random_pages(c, budget, seed=0):
    """Random pages of every sequence, ascending, -1 behind."""
    rnd = random.Random(seed)
    out = torch.full((len(c["lens"]), c["h_kv"], budget), -1, dtype=torch.int32)
    for r, n in enumerate(c["lens"]):
        have = orc.ceil_div(max(0, n), c["page"])
        for h in range(c["h_kv"]):
            mine = sorted(rnd.sample(range(have), min(budget, have)))
            if mine and rnd.random() < 0.7:
                mine[-1] = have - 1          # the page that ends inside a tile, mostly
            out[r, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
    return out


def _attend(c, pages, lse=True, out=None, **other):
    a = {n: _cu(other.get(n, c[n])) for n in ("q", "k", "v", "table")}
    o = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device="cuda") if out is None else out
    s = torch.full(c["q"].shape[:2], 7.0, device="cuda") if lse else None
    _ps().paged_sparse_decode(o, a["q"], a["k"], a["v"], a["table"], _lens(c), pages.cuda(), c["scale"], c["name"],
                              _cu(c["ks"]), _cu(c["vs"]), out_lse=s)
    return o, s


def _check_attend(c, pages, got, lse):
    want, tol, wl, tl = orc.sparse_ref(c["q"], c["k"], c["v"], c["table"], c["lens"], pages, c["scale"], c["ks"], c["vs"])
    _hold(got, want, tol, "out")
    _hold(lse, wl, tl, "lse")
    return want


@pytest.mark.parametrize("kv", ["bf16", "f16", "fp8"])
@pytest.mark.parametrize("d, h_kv, group, page, budget, layout", [
    (64, 2, 4, 16, 6, "hnd"), (128, 8, 4, 16, 12, "nhd"), (128, 1, 16, 32, 5, "hnd"), (256, 2, 7, 16, 9, "nhd"),
    (64, 1, 1, 48, 1, "hnd"), (256, 1, 12, 16, 40, "hnd"), (128, 2, 8, 272, 3, "nhd"), (128, 3, 3, 16, 70, "hnd")])
def test_paged_sparse_decode(kv, d, h_kv, group, page, budget, layout):
    lens = [1, 0, page, 7 * page + 3, 40 * page + 1 if page < 100 else 5 * page + 1, 16 * page - 1 if page < 100 else 31]
    c = _cache_case(lens, d=d, h_kv=h_kv, group=group, page=page, kv=kv, layout=layout, seed=d + group)
    pages = _random_pages(c, budget, seed=group)
    got, lse = _attend(c, pages)
    _check_attend(c, pages, got, lse)
    assert (got[1] == 0).all() and torch.isneginf(lse[1]).all()


@pytest.mark.parametrize("rows, budget", [(1, 1), (1, 37), (1, 300), (3, 64), (40, 33), (150, 5)])
def test_paged_sparse_decode_however_many_ctas_share_a_row(rows, budget):
    rnd = random.Random(rows)
    c = _cache_case([rnd.randint(1, 320 * 16 if rows < 5 else 600) for _ in range(rows)], d=128, h_kv=2, group=4, seed=rows)
    pages = _random_pages(c, budget)
    got, lse = _attend(c, pages)
    _check_attend(c, pages, got, lse)


def test_paged_sparse_decode_over_every_page_is_the_dense_decode():
    from hk_dsl_b200.ops import paged
    c = _cache_case([1000, 33, 1, 0, 517], d=128, h_kv=2, group=4, seed=9)
    width = c["table"].shape[1]
    pages = torch.arange(width, dtype=torch.int32).expand(5, 2, width).contiguous()       # past the end: none
    got, lse = _attend(c, pages)
    full = torch.empty_like(got)
    paged.paged_attention_decode(full, c["q"].cuda(), c["k"].cuda(), c["v"].cuda(), c["table"].cuda(), _lens(c), c["scale"])
    want, tol, _, _ = orc.sparse_ref(c["q"], c["k"], c["v"], c["table"], c["lens"], pages, c["scale"])
    _hold(got, want, tol)
    _hold(full, got.double().cpu(), 2 * tol)


def test_paged_sparse_decode_list_entries():
    """Negative entries anywhere, pages past the sequence or the table, an unordered list, a page twice, a list of none."""
    c = _cache_case([300, 300, 300, 300], d=64, h_kv=1, group=4, seed=11)
    w = c["table"].shape[1]
    pages = torch.tensor([[-1, 5, -1, 2, 18], [18, 18, 0, 3, 3], [w, 2 ** 30, 19, -2 ** 31, 2 ** 31 - 1], [7, -1, -1, -1, 40]],
                         dtype=torch.int32).view(4, 1, 5)
    got, lse = _attend(c, pages)
    want = _check_attend(c, pages, got, lse)
    assert (want[2] == 0).all() and (got[2] == 0).all()
    got0, lse0 = _attend(c, torch.empty(4, 1, 0, dtype=torch.int32))
    assert (got0 == 0).all() and torch.isneginf(lse0).all()


def test_paged_sparse_decode_strides_and_rows_left_alone():
    c = _cache_case([100, 37], d=64, h_kv=2, group=2, seed=12)
    pages = _random_pages(c, 3)
    q = torch.randn(2, 5, 96, device="cuda").to(BF)[:, :4, 16:80]
    q.copy_(c["q"])
    store = torch.full((4, 6, 72), 3.0, dtype=BF, device="cuda")
    out = store[1:3, :4, 4:68]
    kv = torch.zeros(c["k"].shape[0], 16, 2, 2 * 64, dtype=BF, device="cuda")      # K and V side by side
    k, v = kv[..., :64], kv[..., 64:]
    k.copy_(c["k"]); v.copy_(c["v"])
    listed = torch.full((2, 2, 9), 1, dtype=torch.int32)
    listed[:, :, :3] = pages
    table = torch.zeros(2, 2 * c["table"].shape[1], dtype=torch.int32)
    table[:, :c["table"].shape[1]] = c["table"]
    lse = torch.empty(2, 4, device="cuda")
    _ps().paged_sparse_decode(out, q, k, v, table.cuda()[:, :c["table"].shape[1]], _lens(c), listed.cuda()[:, :, :3], c["scale"],
                              out_lse=lse)
    _check_attend(c, pages, out, lse)
    keep = store.clone(); keep[1:3, :4, 4:68] = 3.0
    assert (keep == 3.0).all()


def test_paged_sparse_decode_shows_a_broken_key_and_an_extreme_one():
    c = _cache_case([64, 64, 64], d=64, h_kv=1, group=2, seed=13, nan_tail=False)
    k = c["k"]
    k[int(c["table"][0, 1]), 3, 0, 5] = float("nan")
    k[int(c["table"][1, 1])] = torch.finfo(BF).min                 # logits near the type's lowest value
    pages = torch.arange(4, dtype=torch.int32).expand(3, 1, 4).contiguous()
    got, lse = _attend(c, pages)
    assert torch.isnan(got[0]).all() and torch.isnan(lse[0]).all()
    want, tol, wl, tl = orc.sparse_ref(c["q"][2:], k, c["v"], c["table"][2:], c["lens"][2:], pages[2:], c["scale"])
    _hold(got[2:], want, tol)
    # row 1: that page's products are 3.39e38 |q_d|, past fp32's 3.40e38 wherever |q_d| > 1.004, with both signs among
    # them; logits outside fp32 are no numbers. They show as NaN, or, all of them -inf, as pages without weight.
    assert (c["q"][1].abs() > 1.004).any(-1).all()
    rest = torch.tensor([[0, 2, 3]], dtype=torch.int32).view(1, 1, 3)
    want, tol, _, _ = orc.sparse_ref(c["q"][1:2], k, c["v"], c["table"][1:2], c["lens"][1:2], rest, c["scale"])
    for h in range(2):
        if not torch.isnan(got[1, h]).all():
            _hold(got[1, h], want[0, h], tol[0, h])


# ------------------------------------------------------------------------------ together

class _Loop:
    """A small serving loop's device state, and its step as a user writes it."""

    def __init__(self, n, h_kv=2, group=4, d=64, page=16, width=16, pool=150, rows=160, budget=6, kv="bf16"):
        from hk_dsl_b200.ops import paged
        ps = _ps()
        self.paged, self.ps, self.page, self.d, self.n, self.rows = paged, ps, page, d, n, rows
        dev = dict(device="cuda")
        act = F16 if kv == "f16" else BF
        self.act, self.name = act, "fp8" if kv == "fp8" else "auto"
        store = F8 if kv == "fp8" else act
        self.k = torch.zeros(pool, h_kv, page, d, **dev).to(store).transpose(1, 2)
        self.v = torch.zeros(pool, h_kv, page, d, **dev).to(store).transpose(1, 2)
        self.ks = torch.tensor([0.0125], **dev) if kv == "fp8" else None
        self.bounds = ps.page_bounds(self.k)
        i32 = dict(dtype=torch.int32, **dev)
        self.table, self.lens, self.new = torch.zeros(n, width, **i32), torch.zeros(n, **i32), torch.zeros(n, **i32)
        self.free = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.count = torch.tensor([pool], **i32)
        self.slots, self.pos = torch.zeros(rows, dtype=torch.int64, **dev), torch.zeros(rows, dtype=torch.int64, **dev)
        self.starts, self.status = torch.zeros(n + 1, **i32), torch.zeros(n, **i32)
        self.key = torch.zeros(rows, h_kv, d, dtype=act, **dev)
        self.value = torch.zeros(rows, h_kv, d, dtype=act, **dev)
        self.q = torch.zeros(n, h_kv * group, d, dtype=act, **dev)
        self.scores = torch.zeros(n, h_kv, width, **dev)
        self.pages = torch.zeros(n, h_kv, budget, **i32)
        self.out, self.lse = torch.zeros_like(self.q), torch.zeros(n, h_kv * group, **dev)
        self.h_kv, self.scale = h_kv, d ** -0.5

    def fill(self, seed, new):
        g = torch.Generator().manual_seed(seed)
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        for t in (self.key, self.value, self.q):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))

    def step(self):
        ps, p = self.ps, self.paged
        ps.advance_tables(self.table, self.lens, self.new, self.free, self.count, self.page, self.slots, self.pos, self.starts,
                          self.status)
        p.reshape_and_cache(self.key, self.value, self.k, self.v, self.slots, self.name, self.ks, self.ks)
        ps.update_page_bounds(self.bounds, self.k, self.table, self.lens, self.starts, num_tokens=self.rows)
        ps.page_scores(self.scores, self.q, self.bounds, self.table, self.lens, self.scale, self.page, self.name, self.ks)
        ps.select_pages(self.pages, self.scores, self.lens, self.page, first=1, last=2)
        ps.paged_sparse_decode(self.out, self.q, self.k, self.v, self.table, self.lens, self.pages, self.scale, self.name,
                               self.ks, self.ks, out_lse=self.lse)

    def check(self, model):
        """Against `model`: per request the rows written so far, kept apart from the cache and its pages."""
        torch.cuda.synchronize()
        lens = self.lens.tolist()
        assert lens == [len(m) for m in model]
        c = lambda t: t.cpu()  # noqa: E731
        k, v, table = c(self.k), c(self.v), c(self.table)
        for i, m in enumerate(model):
            for j, (key, value) in enumerate(m):
                b = int(table[i, j // self.page])
                assert _same(k[b, j % self.page], key) and _same(v[b, j % self.page], value)
        ks = c(self.ks) if self.ks is not None else None
        every = orc.bounds_ref(c(self.bounds), k, table, lens, _cum(lens))
        assert _same(self.bounds, every)             # each live page's summary is of what it holds
        want, tol = orc.scores_ref(c(self.q), every, table, lens, self.page, self.scale, ks)
        _hold(self.scores, want, tol, "scores")
        assert torch.equal(c(self.pages), orc.select_ref(c(self.scores), lens, self.page, self.pages.shape[2], 1, 2))
        want, tol, wl, tl = orc.sparse_ref(c(self.q), k, v, table, lens, c(self.pages), self.scale, ks, ks)
        _hold(self.out, want, tol, "out")
        _hold(self.lse, wl, tl, "lse")

    def rows_of(self, i):
        s = self.starts.tolist()
        for t in range(s[i], s[i + 1]):
            key, value = self.key[t].cpu(), self.value[t].cpu()
            if self.ks is not None:
                key, value = dense.quantize_fp8(key, self.ks.cpu()), dense.quantize_fp8(value, self.ks.cpu())
            yield key, value

    def follow(self, model, new):
        for i, n in enumerate(new):
            if int(self.status[i]):
                continue
            if n >= 0:
                model[i].extend(self.rows_of(i))
            else:
                del model[i][max(0, len(model[i]) + n):]


def _cum(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + max(0, n))
    return s


STEPS = [[70, 33, 0, 1, 16], [1, 1, 50, 1, 1], [1, 1, 1, -1, 1], [1, -20, 1, 3, 15], [-500, 1, 1, 1, 1], [90, 1, 1, 1, -16],
         [1, 1, 1, 0, 1], [120, 100, 1, 1, 1]]


@pytest.mark.parametrize("kv", ["bf16", "f16", "fp8"])
def test_a_serving_loop(kv):
    """Prompts, decoding, dropped drafts, a finished request and its successor, a refused one: the step as it is used."""
    s = _Loop(5, kv=kv)
    model = [[] for _ in range(5)]
    for i, new in enumerate(STEPS):
        s.fill(i, new)
        s.step()
        s.follow(model, new)
        s.check(model)
    assert int(s.status[0]) == 0 and s.status.tolist()[1] == orc.NO_ROWS       # 120 + 100 rows of 160


def test_a_captured_step_replays_over_new_requests():
    s = _Loop(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.fill(0, [0] * 5)
        s.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step()
    model = [[] for _ in range(5)]
    for i, new in enumerate(STEPS):
        s.fill(i, new)
        graph.replay()
        s.follow(model, new)
        s.check(model)


def test_two_steps_at_once_on_two_streams():
    """No call keeps anything of its own: two loops in flight together answer as each does alone."""
    alone = []
    for seed in (0, 1):
        s = _Loop(5)
        s.fill(seed, STEPS[0])
        for _ in range(3):
            s.step()
        alone.append((s.out.clone(), s.pages.clone(), s.slots.clone()))
    loops, streams = [_Loop(5), _Loop(5)], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed, s in enumerate(loops):
        s.fill(seed, STEPS[0])
    torch.cuda.synchronize()
    for _ in range(3):
        for s, st in zip(loops, streams):
            with torch.cuda.stream(st):
                s.step()
    torch.cuda.synchronize()
    for s, (out, pages, slots) in zip(loops, alone):
        assert torch.equal(s.out, out) and torch.equal(s.pages, pages) and torch.equal(s.slots, slots)


def test_fp8_bytes_in_uint8_storage():
    c = _cache_case([200, 77], d=128, h_kv=2, group=4, kv="fp8", seed=31)
    pages = _random_pages(c, 7)
    b = _bounds_of(c)
    got, lse = _attend(c, pages)
    raw, rlse = _attend(c, pages, k=c["k"].view(torch.uint8), v=c["v"].view(torch.uint8))
    assert torch.equal(got, raw) and torch.equal(lse, rlse)
    s = [torch.empty(2, 2, c["table"].shape[1], device="cuda") for _ in range(2)]
    for t, bb in zip(s, (b, b.view(torch.uint8))):
        _ps().page_scores(t, c["q"].cuda(), bb.cuda(), c["table"].cuda(), _lens(c), c["scale"], 16, "fp8", c["ks"].cuda())
    assert torch.equal(s[0], s[1])


def test_answers_over_disjoint_pages_merge():
    """Two selections' answers, folded by their sum-exps, are the answer over both."""
    from hk_dsl_b200.ops import paged
    c = _cache_case([700, 90, 0], d=128, h_kv=2, group=4, seed=41)
    every = torch.arange(c["table"].shape[1], dtype=torch.int32).expand(3, 2, -1).contiguous()
    parts = [_attend(c, every[:, :, i::2].contiguous()) for i in range(2)]
    out = torch.empty(3, 8, 128, dtype=BF, device="cuda")
    paged.merge_partials(out, torch.stack([p[0].float() for p in parts]), torch.stack([p[1] for p in parts]))
    want, tol, _, _ = orc.sparse_ref(c["q"], c["k"], c["v"], c["table"], c["lens"], every, c["scale"])
    # each part's own bounds (its rounding to bf16 among them), weighted, then one more rounding
    part_tol = [orc.sparse_ref(c["q"], c["k"], c["v"], c["table"], c["lens"], every[:, :, i::2], c["scale"])[:3] for i in range(2)]
    l = torch.stack([p[2] for p in part_tol])
    w = torch.exp(l - torch.logsumexp(l, 0)).nan_to_num(0.0)
    _hold(out, want, sum(w[i].unsqueeze(-1) * part_tol[i][1] for i in range(2)) * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8 + 2.0 ** -16)


def test_a_step_without_new_rows_summarises_shortened_pages_again():
    c = _cache_case([40, 21], d=64, h_kv=1, seed=51)
    b = _bounds_of(c).cuda()
    c["lens"] = [35, 5]
    _ps().update_page_bounds(b, c["k"].cuda(), c["table"].cuda(), _lens(c), torch.zeros(3, dtype=torch.int32, device="cuda"), num_tokens=0)
    want = orc.bounds_ref(_bounds_of(dict(c, lens=[40, 21])), c["k"], c["table"], [35, 5], [0, 0, 0])
    assert _same(b, want)


def test_the_torch_ops_are_the_calls():
    from hk_dsl_b200.runtime import torch_ext
    torch_ext.sparse_ops()
    hk = torch.ops.hk
    a, b = _Loop(5), _Loop(5)
    for s in (a, b):
        s.fill(0, STEPS[0])
    a.step()
    assert hk.advance_tables(b.table, b.lens, b.new, b.free, b.count, b.page, b.slots, b.pos, b.starts, b.status) is None
    b.paged.reshape_and_cache(b.key, b.value, b.k, b.v, b.slots)
    hk.update_page_bounds(b.bounds, b.k, b.table, b.lens, b.starts, b.rows)
    hk.page_scores(b.scores, b.q, b.bounds, b.table, b.lens, b.scale, b.page, "auto", None)
    hk.select_pages(b.pages, b.scores, b.lens, b.page, 1, 2)
    hk.paged_sparse_decode(b.out, b.q, b.k, b.v, b.table, b.lens, b.pages, b.scale, "auto", None, None, b.lse)
    for name in ("table", "lens", "free", "count", "slots", "pos", "starts", "status", "scores", "pages", "out", "lse"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_a_call_behind_another_streams_event_sees_its_writes():
    """The kernels may take their places while the one before in their stream still runs; what else the stream waits for
    comes first all the same: another stream's event, a copy, an ordinary kernel."""
    c = _cache_case([600, 333], d=128, h_kv=2, group=4, seed=61)
    pages = _random_pages(c, 9)
    want, _ = _attend(c, pages)
    k, v, table, lens, pg = c["k"].cuda(), c["v"].cuda(), c["table"].cuda(), _lens(c), pages.cuda()
    good, host = c["q"].cuda(), c["q"].pin_memory()
    q, out = torch.zeros_like(good), torch.empty_like(good)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def call():
        _ps().paged_sparse_decode(out, q, k, v, table, lens, pg, c["scale"])

    for how in ("event", "copy", "kernel", "event", "kernel"):
        q.zero_(); out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(two):
            call()                                    # the call in front: over the old query
            if how == "event":
                with torch.cuda.stream(one):
                    torch.cuda._sleep(20_000_000)     # some 10 ms
                    q.copy_(good)
                    done = one.record_event()
                two.wait_event(done)
            elif how == "copy":
                q.copy_(host, non_blocking=True)
            else:
                torch.cuda._sleep(2_000_000)
                q.add_(good)
            call()
            answer = out.clone()                      # an ordinary kernel behind it
        torch.cuda.synchronize()
        assert torch.equal(answer, want), how


def test_the_same_call_twice_gives_the_same_bits():
    c = _cache_case([4000, 900, 31], d=128, h_kv=2, group=4, seed=21)
    pages = _random_pages(c, 60)
    a, la = _attend(c, pages)
    b, lb = _attend(c, pages)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_a_page_pool_past_four_gigabytes():
    """Offsets of pages that lie past 2^32 bytes of the cache."""
    page, d, h_kv = 16, 128, 8
    nb = 2 ** 32 // (page * d * h_kv * 2) + 40
    k = torch.zeros(nb, h_kv, page, d, dtype=BF, device="cuda").transpose(1, 2)
    v = torch.zeros(nb, h_kv, page, d, dtype=BF, device="cuda").transpose(1, 2)
    ids = torch.tensor([[nb - 1, nb - 2, 0, nb - 7, nb // 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    for b in ids[0].tolist():
        k[b] = torch.randn(page, h_kv, d, generator=g).to(BF).cuda()
        v[b] = torch.randn(page, h_kv, d, generator=g).to(BF).cuda()
    q = torch.randn(1, 32, d, generator=g).to(BF)
    lens = torch.tensor([5 * page - 3], dtype=torch.int32)
    pages = torch.tensor([0, 3, 4], dtype=torch.int32).expand(1, h_kv, 3).contiguous()
    bounds = torch.zeros_like(_ps().page_bounds(k))
    _ps().update_page_bounds(bounds, k, ids.cuda(), lens.cuda(), torch.tensor([0, 77], dtype=torch.int32).cuda(), num_tokens=77)
    scores = torch.zeros(1, h_kv, 5, device="cuda")
    _ps().page_scores(scores, q.cuda(), bounds, ids.cuda(), lens.cuda(), d ** -0.5, page)
    out = torch.zeros(1, 32, d, dtype=BF, device="cuda")
    _ps().paged_sparse_decode(out, q.cuda(), k, v, ids.cuda(), lens.cuda(), pages.cuda(), d ** -0.5)
    small = torch.arange(5, dtype=torch.int32).view(1, 5)
    ks, vs = k[ids[0].long().cuda()].cpu(), v[ids[0].long().cuda()].cpu()
    b = orc.bounds_ref(torch.zeros(5, h_kv, 2, d, dtype=BF), ks, small, lens.tolist(), [0, 77])
    assert _same(bounds[ids[0].long().cuda()], b)
    want, tol = orc.scores_ref(q, b, small, lens.tolist(), page, d ** -0.5)
    _hold(scores, want, tol)
    want, tol, _, _ = orc.sparse_ref(q, ks, vs, small, lens.tolist(), pages, d ** -0.5)
    _hold(out, want, tol)
