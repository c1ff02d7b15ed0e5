"""Decode over selected pages: what the host refuses, before any launch and without a GPU, and the oracle's own rules."""

import os
import random
import re

import pytest
import torch

from hk_dsl_b200.ops import paged_sparse as ps
from hk_dsl_b200.runtime import lib
from oracle import sparse_oracle as orc

I32, I64 = torch.int32, torch.int64


def _z(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def _tables(**other):
    a = dict(block_tables=_z(3, 4), seq_lens=_z(3), new_tokens=_z(3), free_pages=_z(8), free_count=_z(1), block_size=16,
             slot_mapping=_z(5, dtype=I64), positions=_z(5, dtype=I64), query_start_loc=_z(4), status=_z(3))
    a.update(other)
    return a


@pytest.mark.parametrize("other, error", [
    (dict(block_tables=_z(3, 4, dtype=I64)), TypeError), (dict(block_tables=_z(12)), TypeError),
    (dict(block_tables=_z(4, 3).t()), TypeError), (dict(block_tables=_z(2, 4)), ValueError),
    (dict(block_tables=_z(1, 4).expand(3, 4)), ValueError),
    (dict(seq_lens=_z(3, dtype=I64)), TypeError), (dict(seq_lens=_z(6)[::2]), TypeError), (dict(new_tokens=_z(2)), ValueError),
    (dict(new_tokens=_z(3, dtype=torch.float32)), TypeError), (dict(free_pages=_z(8, dtype=I64)), TypeError),
    (dict(free_count=_z(0)), ValueError), (dict(slot_mapping=_z(5)), TypeError), (dict(positions=_z(4, dtype=I64)), ValueError),
    (dict(query_start_loc=_z(3)), ValueError), (dict(status=_z(2)), ValueError), (dict(), RuntimeError),
])
def test_advance_tables_refuses(other, error):
    with pytest.raises(error, match="hk.ops"):
        ps.advance_tables(**_tables(**other))


def _attn(**other):
    bf = torch.bfloat16
    a = dict(out=_z(2, 8, 64, dtype=bf), query=_z(2, 8, 64, dtype=bf), key_cache=_z(5, 16, 2, 64, dtype=bf),
             value_cache=_z(5, 16, 2, 64, dtype=bf), block_tables=_z(2, 3), seq_lens=_z(2), pages=_z(2, 2, 3), scale=0.1)
    a.update(other)
    return a


@pytest.mark.parametrize("other, error", [
    (dict(query=_z(2, 8, 64, dtype=torch.float32)), ValueError), (dict(query=_z(2, 512, dtype=torch.bfloat16)), ValueError),
    (dict(out=_z(2, 8, 64, dtype=torch.float16)), ValueError), (dict(out=_z(3, 8, 64, dtype=torch.bfloat16)), ValueError),
    (dict(key_cache=_z(5, 16, 2, 128, dtype=torch.bfloat16)), ValueError),
    (dict(value_cache=_z(5, 16, 2, 64, dtype=torch.float16)), ValueError),
    (dict(key_cache=_z(5, 16, 64, 2, dtype=torch.bfloat16).transpose(2, 3)), ValueError),
    (dict(block_tables=_z(1, 3)), ValueError), (dict(seq_lens=_z(1)), ValueError), (dict(pages=_z(2, 1, 3)), ValueError),
    (dict(pages=_z(2, 2, 3, dtype=I64)), TypeError), (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(out_lse=_z(2, 8, dtype=torch.bfloat16)), ValueError), (dict(out_lse=_z(2, 7, dtype=torch.float32)), ValueError),
    (dict(kv_cache_dtype="fp8"), TypeError), (dict(kv_cache_dtype="int4"), NotImplementedError), (dict(), RuntimeError),
])
def test_paged_sparse_decode_refuses(other, error):
    with pytest.raises(error, match="hk.ops"):
        ps.paged_sparse_decode(**_attn(**other))


def test_scores_select_and_bounds_refuse():
    bf = torch.bfloat16
    cache, bounds, table, lens = _z(5, 16, 2, 64, dtype=bf), _z(5, 2, 2, 64, dtype=bf), _z(2, 3), _z(2)
    q, scores = _z(2, 8, 64, dtype=bf), _z(2, 2, 3, dtype=torch.float32)
    assert ps.page_bounds(cache).shape == bounds.shape and ps.page_bounds(cache).dtype == bf
    for bad in (_z(5, 2, 64, dtype=bf), _z(5, 2, 3, 64, dtype=bf), _z(5, 2, 64, 2, dtype=bf).transpose(2, 3),
                _z(5, 2, 2, 64, dtype=torch.float16), _z(5, 4, 2, 64, dtype=bf)):
        with pytest.raises(ValueError, match="bounds"):
            ps.update_page_bounds(bad, cache, table, lens)
    with pytest.raises(TypeError, match="float32"):
        ps.update_page_bounds(bounds.float(), cache.float(), table, lens)
    with pytest.raises(ValueError, match="num_tokens"):
        ps.update_page_bounds(bounds, cache, table, lens, _z(3))
    with pytest.raises(ValueError, match="query_start_loc"):
        ps.update_page_bounds(bounds, cache, table, lens, _z(2), num_tokens=4)
    with pytest.raises(ValueError, match="bounds"):
        ps.page_scores(scores, q[:, :, :32], bounds, table, lens, 1.0, 16)
    with pytest.raises(ValueError, match="scores"):
        ps.page_scores(scores[:, :, :2], q, bounds, table, lens, 1.0, 16)
    with pytest.raises(ValueError, match="scores"):
        ps.page_scores(scores.double(), q, bounds, table, lens, 1.0, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ps.page_scores(scores, q, bounds, table, lens, 1.0, 16)
    with pytest.raises(ValueError, match="budget"):
        ps.select_pages(_z(2, 2, 4), scores, lens, 16, first=1, last=4)
    with pytest.raises(ValueError, match="scores"):
        ps.select_pages(_z(2, 1, 8), scores, lens, 16)
    with pytest.raises(ValueError, match="lengths"):
        ps.select_pages(_z(2, 2, 8), scores, lens[:1], 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ps.select_pages(_z(2, 2, 8), scores, lens, 16)


def test_the_c_entries_refuse_before_any_launch():
    l = lib.load()

    def adv(width=4, stride=4, lens=16, n=3, page=16, cap=8, count=16, slots=16, rows=5, starts=16):
        return l.hkb_advance_tables(lib.ADVANCE(16, stride, width, lens, 16, n, page, 16, cap, count, slots, 16, rows, starts, 16), None)

    assert adv(n=-1) == adv(rows=-1) == adv(cap=-1) == adv(cap=2 ** 31) == adv(width=2 ** 31) == adv(rows=2 ** 31) == -9
    assert adv(page=0) == -3 and adv(stride=3) == -6
    assert adv(lens=0) == adv(count=0) == adv(slots=0) == adv(starts=0) == -1

    def bnd(b=16, sb=256, sk=128, n=2, tok=4, hkv=1, d=128, page=16, dt=0, starts=0):
        return l.hkb_page_bounds(lib.PAGE_BOUNDS(b, sb, 256, 4, 16, 2048, sk, 32768, 4, 16, 4, 4, 16, starts, n, tok, hkv, d, page, dt), None)

    assert bnd(n=0) == 0
    assert bnd(n=-1) == bnd(hkv=0) == bnd(tok=-1) == bnd(n=2 ** 31) == -9 and bnd(b=0) == -1
    assert bnd(d=96) == -2 and bnd(page=0) == -3 and bnd(dt=7) == -5
    assert bnd(sb=252) == bnd(sk=124) == -6 and bnd(b=24) == -7

    def sco(s=16, cols=8, q=16, qs=512, nb=4, rows=2, hq=4, hkv=2, d=128, page=16, dt=0, ks=0):
        return l.hkb_page_scores(lib.PAGE_SCORES(s, 16, 8, cols, q, qs, 128, 16, 512, 256, nb, 16, 8, 16, rows, hq, hkv, d, page,
                                                 dt, ks, 0.1), None)

    assert sco(rows=0) == 0 and sco(cols=0) == 0
    assert sco(rows=-1) == sco(rows=65536) == sco(nb=0) == sco(cols=2 ** 31) == -9 and sco(s=0) == -1
    assert sco(d=96) == -2 and sco(page=0) == -3 and sco(hq=3) == sco(hq=34) == -4
    assert sco(dt=3) == -5 and sco(dt=1) == -10 and sco(qs=508) == -6 and sco(q=8) == sco(s=18) == -7

    def sel(p=16, budget=8, s=16, cols=20, rows=2, hkv=2, page=16, first=1, last=4):
        return l.hkb_select_pages(lib.SELECT_PAGES(p, 16, 8, budget, s, 40, 20, cols, 16, rows, hkv, page, first, last), None)

    assert sel(rows=0) == 0 and sel(budget=0, first=0, last=0) == 0
    assert sel(rows=-1) == sel(budget=4) == sel(first=-1) == sel(rows=2 ** 30) == sel(hkv=65536) == -9 and sel(p=0) == sel(s=0) == -1
    assert sel(page=0) == -3 and sel(p=18) == -7

    def att(out=16, os=512, lse=0, q=16, sk=128, nb=4, table=16, pages=16, budget=4, rows=2, hq=4, hkv=2, d=128, page=16, dt=0, ks=0):
        return l.hkb_paged_sparse_decode(lib.SPARSE_DECODE(
            out, os, 128, lse, q, 512, 128, 16, 2048, sk, 32768, nb, 16, 2048, 128, 32768, 4, table, 8, 8, 16, pages, 8, 4, budget,
            rows, hq, hkv, d, page, dt, ks, 0, 0.1), None)

    assert att(rows=0) == 0
    assert att(rows=-1) == att(rows=65536) == att(budget=-1) == att(nb=0) == -9 and att(budget=2 ** 31 - 1, page=32) == -9
    assert att(out=0) == att(q=0) == att(table=0) == att(pages=0) == -1
    assert att(d=96) == -2 and att(page=24) == -3 and att(hq=3) == att(hq=34) == -4 and att(dt=9) == -5
    assert att(dt=1) == att(dt=1, ks=16) == -10
    assert att(os=510) == att(sk=124) == -6 and att(out=20) == att(lse=18) == att(q=8) == -7
    for fn in ("hkb_advance_tables", "hkb_page_bounds", "hkb_page_scores", "hkb_select_pages", "hkb_paged_sparse_decode"):
        assert getattr(l, fn)(None, None) == -1


def test_the_argument_structs_are_packed_as_the_header_declares_them():
    """One 64-bit word a field, in the header's order; hkb_cache_t is five words."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "hkb.h")).read()
    for struct, pack in (("hkb_advance_t", lib.ADVANCE), ("hkb_page_bounds_t", lib.PAGE_BOUNDS),
                         ("hkb_page_scores_t", lib.PAGE_SCORES), ("hkb_select_pages_t", lib.SELECT_PAGES),
                         ("hkb_sparse_decode_t", lib.SPARSE_DECODE)):
        body = re.search(r"typedef struct \{([^}]*)\} " + struct, text).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        words, doubles = 0, []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            each = 5 if decl.startswith("hkb_cache_t") else 1
            assert each == 5 or "*" in decl or decl.startswith(("int64_t", "double")), decl
            doubles += [decl.startswith("double")] * (each * (decl.count(",") + 1))
            words = len(doubles)
        assert len(pack(*[0.0 if d else 0 for d in doubles])) == 8 * words, struct
        assert not any(doubles[:-1])


def test_the_oracles_tables_keep_every_page():
    """Whatever a random run of steps asks for, a page is free or one request's, never both, and every token's slot
    is in its request's page."""
    rnd = random.Random(3)
    page, width, pool, n = 4, 6, 30, 7
    table, lens = [[0] * width for _ in range(n)], [0] * n
    free, count = rnd.sample(range(pool), pool), pool
    for _ in range(200):
        new = [rnd.choice([0, 1, 1, 5, 13, -1, -3, -100]) for _ in range(n)]
        old, was = list(lens), count
        table, lens, free, count, slots, positions, starts, status = orc.advance_ref(table, lens, new, free, count, page, 25)
        owned = [p for r, m in zip(table, lens) for p in r[:orc.ceil_div(m, page)]]
        assert sorted(owned + free[:count]) == list(range(pool))
        for i in range(n):
            assert lens[i] == (max(0, old[i] + new[i]) if status[i] == orc.OK else old[i])
            for j in range(max(0, new[i])):
                t = starts[i] + j
                if status[i] == orc.OK:
                    assert positions[t] == old[i] + j
                    assert slots[t] == table[i][positions[t] // page] * page + positions[t] % page
                elif t < 25:
                    assert slots[t] == -1
        assert was >= 0


def test_the_oracles_selection_matches_a_stable_sort():
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 6, (3, 2, 40), generator=g).float()
    got = orc.select_ref(x, [16 * 40, 16 * 33 + 1, 16 * 3], 16, 9, 1, 2)
    for r, n in ((0, 40), (1, 34)):
        for h in range(2):
            key = x[r, h, :n].clone()
            key[:1] = key[n - 2:] = 100.0
            best = torch.sort(key, descending=True, stable=True).indices[:9].sort().values
            assert got[r, h].tolist() == best.tolist()
    assert got[2, 0].tolist() == [0, 1, 2] + [-1] * 6
