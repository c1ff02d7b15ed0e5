"""Decode over selected pages of the paged KV cache, and the page bookkeeping under it: the host side.

A long context's decode step need not read the whole cache. `update_page_bounds` keeps a summary of every page (the
least and the greatest key of each channel), `page_scores` bounds from the summaries the best logit a query can have
in a page, `select_pages` takes the budget's best pages of every query row and kv head, and `paged_sparse_decode`
attends to those alone. `advance_tables` builds what all of them read -- block tables, slot mapping, positions -- on
the GPU from the requests' lengths. A step of a layer:

    advance_tables(block_tables, seq_lens, new_tokens, free_pages, free_count, block_size, slots, positions, starts, status)
    reshape_and_cache(key, value, key_cache, value_cache, slots)                     # hk_dsl_b200.ops.paged
    update_page_bounds(bounds, key_cache, block_tables, seq_lens)
    page_scores(scores, query, bounds, block_tables, seq_lens, scale, block_size)
    select_pages(pages, scores, seq_lens, block_size)
    paged_sparse_decode(out, query, key_cache, value_cache, block_tables, seq_lens, pages, scale)

Caches, queries and tables are those of `hk_dsl_b200.ops.paged`: `(blocks, block_size, kv_heads, head_dim)` views of any
strides in bf16, fp16 or fp8-e4m3, `(rows, q_heads, head_dim)` queries, int32 tables and lengths, row i of the query
belonging to row i of the table. Every call is one launch on torch's current stream; it allocates nothing, reads
nothing back and can be captured into a CUDA graph. A tensor that a call writes overlaps neither itself (`expand`) nor
another one of the call's; a page is read by as many rows as list it. There is no fallback: a call the kernels do not
take raises.
"""

from __future__ import annotations

from typing import Optional

import torch

from ..runtime import lib as _lib
from .paged import _FP8_DTYPES, _need_cuda, _scale_ptr, kv_dtype_code

#: `status` of `advance_tables`
REQ_OK, REQ_NO_PAGES, REQ_TABLE_FULL, REQ_NO_ROWS = 0, 1, 2, 3

_WHO = "hk.ops.paged_sparse"
_I32, _I64, _F32, _BF16, _F16 = torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.float16

# A decode step makes a handful of these calls a layer, each a few microseconds on the GPU, so what the host spends on a
# call counts. Tensors' sizes and strides are read once a call, devices by number, and the stream's handle is taken
# straight from torch's binding where it has one (2.3 us a call through torch.cuda.current_stream, 0.1 us so).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The current stream's handle, where every tensor is on the current CUDA device; else what `_need_cuda` raises."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            break
    else:
        if dev >= 0 and dev == torch.cuda.current_device():
            return _raw_stream(dev)
    _need_cuda(first, *others)
    raise RuntimeError(f"{_WHO}: tensors on different devices")


def _index(name: str, t: torch.Tensor, dim: int, dtype=_I32) -> None:
    """An index tensor: `dim` axes, the last one contiguous."""
    if t.dtype is not dtype or t.dim() != dim or not (t.is_contiguous() or t.shape[-1] <= 1 or t.stride(-1) == 1):
        raise TypeError(f"{_WHO}: {name} is {tuple(t.shape)} {t.dtype} strides {tuple(t.stride())}; "
                        f"{dim}-dimensional {dtype} with a contiguous last axis needed")


def _page_size(block_size: int) -> int:
    if block_size < 1:
        raise ValueError(f"{_WHO}: block_size {block_size}: a positive number of tokens")
    return int(block_size)


def _tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, rows: int):
    """The checked table's width and the stride of its rows."""
    shape, strides, lens = block_tables.shape, block_tables.stride(), seq_lens.shape
    if block_tables.dtype is not _I32 or seq_lens.dtype is not _I32 or len(shape) != 2 or strides[1] != 1 \
            or seq_lens.stride() != (1,):
        _index("block_tables", block_tables, 2)       # which of them, and whether it is one the kernels take all the same
        _index("seq_lens", seq_lens, 1)
    have, width = shape
    if have < rows or lens[0] < rows:
        raise ValueError(f"{_WHO}: block_tables {tuple(shape)} and seq_lens {tuple(lens)} for {rows} rows")
    return width, strides[0]


def page_bounds(key_cache: torch.Tensor) -> torch.Tensor:
    """The summary tensor of a key cache: `(blocks, kv_heads, 2, head_dim)` of the cache's type, least keys then
    greatest, uninitialised (`update_page_bounds` fills the pages that it is told of)."""
    nb, _, hkv, d = key_cache.shape
    return torch.empty(nb, hkv, 2, d, device=key_cache.device, dtype=key_cache.dtype)


def advance_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, new_tokens: torch.Tensor,
                   free_pages: torch.Tensor, free_count: torch.Tensor, block_size: int, slot_mapping: torch.Tensor,
                   positions: torch.Tensor, query_start_loc: torch.Tensor, status: torch.Tensor) -> None:
    """Grow or shrink every request by `new_tokens` and write down where its new tokens go; in place, one launch.

    `block_tables` (requests, max_pages) int32 and `seq_lens` (requests,) int32 are the requests as they are;
    `new_tokens` (requests,) int32 what they ask for: a negative number gives tokens back from the end (rejected
    drafts), all of them when the request is finished. `free_pages` (pool,) int32 is a stack whose first `free_count`
    (1,) int32 entries are free pages; new pages come from its top in request order, pages given back go on top of what
    is left, for the next call. Written: `query_start_loc` (requests + 1,) int32, where each request's new tokens begin;
    `slot_mapping` and `positions` (rows,) int64 of every new token in that order, -1 and 0 in the rows behind the last
    one (`reshape_and_cache` skips them, so a captured step may have spare rows); `status` (requests,) int32. A request
    with `REQ_NO_PAGES` (too few free pages; once one is short, so is every later one that needs any), `REQ_TABLE_FULL`
    or `REQ_NO_ROWS` keeps its length, gets no page, and its rows get slot -1. The tokens it asked for are counted in
    `query_start_loc` all the same: behind a `REQ_NO_ROWS` the starts lie past `rows`, and a call that reads query rows by them
    must not be made before `status` was looked at. A page belongs to one request."""
    _index("block_tables", block_tables, 2)
    for t in (seq_lens, new_tokens, free_pages, free_count, query_start_loc, status):
        if t.dtype is not _I32 or t.stride() != (1,):
            for name, x in (("seq_lens", seq_lens), ("new_tokens", new_tokens), ("free_pages", free_pages),
                            ("free_count", free_count), ("query_start_loc", query_start_loc), ("status", status)):
                _index(name, x, 1)
    if slot_mapping.dtype is not _I64 or positions.dtype is not _I64 or slot_mapping.stride() != (1,) or positions.stride() != (1,):
        _index("slot_mapping", slot_mapping, 1, _I64)
        _index("positions", positions, 1, _I64)
    n, = seq_lens.shape
    have, width = block_tables.shape
    stride = block_tables.stride()[0]
    rows, = slot_mapping.shape
    if have < n or new_tokens.shape[0] < n or status.shape[0] < n or query_start_loc.shape[0] < n + 1:
        raise ValueError(f"{_WHO}: {n} requests (seq_lens) with block_tables {tuple(block_tables.shape)}, new_tokens "
                         f"{tuple(new_tokens.shape)}, status {tuple(status.shape)}, query_start_loc "
                         f"{tuple(query_start_loc.shape)} ({n + 1} needed)")
    if free_count.shape[0] < 1 or positions.shape[0] != rows:
        raise ValueError(f"{_WHO}: free_count holds {free_count.numel()} numbers (1 needed); slot_mapping "
                         f"{tuple(slot_mapping.shape)} and positions {tuple(positions.shape)} must be alike")
    if n > 1 and stride < width:
        raise ValueError(f"{_WHO}: block_tables' rows overlap (strides {tuple(block_tables.stride())}); it is written")
    page = _page_size(block_size)
    stream = _on(seq_lens, block_tables, new_tokens, free_pages, free_count, slot_mapping, positions, query_start_loc, status)
    rc = _lib.load().hkb_advance_tables(_lib.ADVANCE(
        block_tables.data_ptr(), stride, width, seq_lens.data_ptr(), new_tokens.data_ptr(), n, page,
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), slot_mapping.data_ptr(), positions.data_ptr(),
        rows, query_start_loc.data_ptr(), status.data_ptr()), stream)
    if rc:
        _lib.check("hkb_advance_tables", rc)


def _kind(cache: torch.Tensor) -> int:
    dtype = cache.dtype
    if dtype is _BF16:
        return _lib.KV_BF16
    if dtype is _F16:
        return _lib.KV_F16
    if dtype not in _FP8_DTYPES:
        raise TypeError(f"{_WHO}: a key cache of {dtype} (bfloat16, float16 and float8_e4m3fn, or uint8 for the latter's "
                        f"bytes, are implemented)")
    return _lib.KV_FP8_E4M3


def _cache_strides(key_cache: torch.Tensor, value_cache: Optional[torch.Tensor] = None):
    """A cache's shape and strides (the value cache's too), checked: head_dim contiguous."""
    shape, ks = key_cache.shape, key_cache.stride()
    vs = value_cache.stride() if value_cache is not None else ks
    if len(shape) != 4 or ks[3] != 1 or vs[-1] != 1 or (value_cache is not None and (
            value_cache.shape != shape or value_cache.dtype is not key_cache.dtype)):
        other = "" if value_cache is None else \
            f" / value_cache {tuple(value_cache.shape)} {value_cache.dtype} strides {tuple(vs)}"
        raise ValueError(f"{_WHO}: key_cache {tuple(shape)} {key_cache.dtype} strides {tuple(ks)}{other}; "
                         f"(blocks, block_size, kv_heads, head_dim) views of one dtype with head_dim contiguous needed")
    return shape, ks, vs


def _bounds_strides(bounds: torch.Tensor):
    shape, strides = bounds.shape, bounds.stride()
    if len(shape) != 4 or shape[2] != 2 or strides[3] != 1 or strides[2] != shape[3]:
        raise ValueError(f"{_WHO}: bounds is {tuple(shape)} strides {tuple(strides)}; "
                         f"(blocks, kv_heads, 2, head_dim) with the last two axes contiguous needed (page_bounds)")
    return shape, strides


def update_page_bounds(bounds: torch.Tensor, key_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                       query_start_loc: Optional[torch.Tensor] = None, *, num_tokens: Optional[int] = None) -> torch.Tensor:
    """Summarise the pages that hold each sequence's newest tokens: `bounds[b, h, 0]` and `[b, h, 1]` become the least
    and the greatest key of every channel over the page's tokens below the sequence's length.

    To be called behind the cache write. Without `query_start_loc` every sequence has one new token; with it (int32,
    sequences + 1, from `advance_tables`) sequence i has `query_start_loc[i + 1] - query_start_loc[i]`, of those that lie
    below `num_tokens`, the step's rows (a host number): the starts run on past it where `advance_tables` refused a
    request for rows. A sequence without new tokens has its last page summarised again: it holds fewer tokens if the
    sequence was shortened. `bounds` is of the cache's type: nothing is rounded. Pages
    are read from the cache as it is, so a call may be repeated; sequences of length 0 are left out. The table has one row a
    sequence (not one a query row, where those are several a sequence): a page that two rows share must be full in both, or
    which of them its summary is of depends on the order."""
    (nb, page, hkv, d), ks, _ = _cache_strides(key_cache)
    bshape, bs = _bounds_strides(bounds)
    code = _kind(key_cache)
    if bounds.dtype is not key_cache.dtype or bshape[1] != hkv or bshape[3] != d:
        raise ValueError(f"{_WHO}: bounds {tuple(bounds.shape)} {bounds.dtype} beside a key cache {tuple(key_cache.shape)} "
                         f"{key_cache.dtype}")
    n = seq_lens.shape[0]
    width, stride = _tables(block_tables, seq_lens, n)
    starts = 0
    if query_start_loc is not None:
        _index("query_start_loc", query_start_loc, 1)
        if query_start_loc.shape[0] < n + 1:
            raise ValueError(f"{_WHO}: query_start_loc has {query_start_loc.shape[0]} entries for {n} sequences")
        if num_tokens is None or num_tokens < 0:
            raise ValueError(f"{_WHO}: query_start_loc needs num_tokens, the rows of the step (a host number), not {num_tokens}")
        starts = query_start_loc.data_ptr()
    stream = _on(bounds, key_cache, block_tables, seq_lens, query_start_loc)
    rc = _lib.load().hkb_page_bounds(_lib.PAGE_BOUNDS(
        bounds.data_ptr(), bs[0], bs[1], bshape[0], key_cache.data_ptr(), ks[0], ks[1], ks[2], nb,
        block_tables.data_ptr(), stride, width, seq_lens.data_ptr(), starts, n, num_tokens or 0, hkv, d,
        page, code), stream)
    if rc:
        _lib.check("hkb_page_bounds", rc)
    return bounds


def _code(kv_cache_dtype: str, cache: torch.Tensor, dtype) -> int:
    """`kv_dtype_code`, the common case first: a 16-bit cache of the query's own type."""
    if kv_cache_dtype == "auto" and cache.dtype is dtype:
        return _lib.KV_BF16 if dtype is _BF16 else _lib.KV_F16
    return kv_dtype_code(kv_cache_dtype, cache, dtype)


def _positive(scale: float) -> float:
    scale = float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError(f"{_WHO}: scale {scale}: a positive number that fp32 holds in full needed (2^-126 to 2^126); the "
                         f"greatest logit is only bounded for a positive one")
    return scale


def _query(query: torch.Tensor):
    """The query's shape and strides, checked."""
    shape, strides, dtype = query.shape, query.stride(), query.dtype
    if len(shape) != 3 or strides[2] != 1 or (dtype is not _BF16 and dtype is not _F16):
        raise ValueError(f"{_WHO}: query is {tuple(shape)} {dtype} strides {tuple(strides)}; "
                         f"(rows, q_heads, head_dim) bfloat16 or float16 with head_dim contiguous needed")
    return shape, strides


def page_scores(scores: torch.Tensor, query: torch.Tensor, bounds: torch.Tensor, block_tables: torch.Tensor,
                seq_lens: torch.Tensor, scale: float, block_size: int, kv_cache_dtype: str = "auto",
                k_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The bound of the best logit every query row can have in every page of its sequence.

    `scores` (rows, kv_heads, max_pages) fp32 gets `scale * k_scale * max_g sum_d max(q_gd low_d, q_gd high_d)`, the
    greatest over the kv head's group of query heads, and -inf for the table's columns behind the sequence.
    `query` (rows, q_heads, head_dim); `bounds` from `update_page_bounds`."""
    (rows, hq, d), qs = _query(query)
    (nb, hkv, _, bd), bs = _bounds_strides(bounds)
    width, stride = _tables(block_tables, seq_lens, rows)
    ss = scores.stride()
    if bd != d or hkv < 1 or hq % hkv:
        raise ValueError(f"{_WHO}: query {tuple(query.shape)} beside bounds {tuple(bounds.shape)}")
    if scores.dtype is not _F32 or scores.shape != (rows, hkv, width) or (width > 1 and ss[2] != 1):
        raise ValueError(f"{_WHO}: scores is {tuple(scores.shape)} {scores.dtype}; ({rows}, {hkv}, {width}) float32 with "
                         f"contiguous columns needed (the table's width)")
    code = _code(kv_cache_dtype, bounds, query.dtype)
    scale, page = _positive(scale), _page_size(block_size)
    stream = _on(query, scores, bounds, block_tables, seq_lens, k_scale)
    rc = _lib.load().hkb_page_scores(_lib.PAGE_SCORES(
        scores.data_ptr(), ss[0], ss[1], width, query.data_ptr(), qs[0], qs[1], bounds.data_ptr(), bs[0], bs[1], nb,
        block_tables.data_ptr(), stride, seq_lens.data_ptr(), rows, hq, hkv, d, page, code,
        _scale_ptr(k_scale, code == _lib.KV_FP8_E4M3, "k_scale") or 0, scale), stream)
    if rc:
        _lib.check("hkb_page_scores", rc)
    return scores


def select_pages(pages: torch.Tensor, scores: torch.Tensor, seq_lens: torch.Tensor, block_size: int, *,
                 first: int = 1, last: int = 4) -> torch.Tensor:
    """The budget's best pages: `pages` (rows, kv_heads, budget) int32 gets, in ascending order and -1 behind, the
    `first` and the `last` pages of the row's sequence and then those of the greatest `scores` (rows, kv_heads, columns)
    fp32, ties to the lowest page, NaN above all numbers. A row with no more pages than the budget gets them all. What the
    columns behind a sequence hold makes no difference.
    The entries number the row's pages (columns of its block table), as `paged_sparse_decode` reads them."""
    pshape, ps, lens = pages.shape, pages.stride(), seq_lens.shape
    if pages.dtype is not _I32 or seq_lens.dtype is not _I32 or len(pshape) != 3 or ps[2] != 1 or seq_lens.stride() != (1,):
        _index("pages", pages, 3)
        _index("seq_lens", seq_lens, 1)
    rows, hkv, budget = pshape
    shape, ss = scores.shape, scores.stride()
    if scores.dtype is not _F32 or len(shape) != 3 or shape[0] != rows or shape[1] != hkv or (shape[2] > 1 and ss[2] != 1):
        raise ValueError(f"{_WHO}: scores is {tuple(shape)} {scores.dtype} beside pages {tuple(pages.shape)}; "
                         f"({rows}, {hkv}, columns) float32 with contiguous columns needed")
    if lens[0] < rows:
        raise ValueError(f"{_WHO}: {lens[0]} lengths for {rows} rows")
    if first < 0 or last < 0 or first + last > budget:
        raise ValueError(f"{_WHO}: first {first} and last {last} pages of a budget of {budget}")
    page = _page_size(block_size)
    stream = _on(pages, scores, seq_lens)
    rc = _lib.load().hkb_select_pages(_lib.SELECT_PAGES(
        pages.data_ptr(), ps[0], ps[1], budget, scores.data_ptr(), ss[0], ss[1], shape[2], seq_lens.data_ptr(), rows, hkv,
        page, first, last), stream)
    if rc:
        _lib.check("hkb_select_pages", rc)
    return pages


def paged_sparse_decode(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                        block_tables: torch.Tensor, seq_lens: torch.Tensor, pages: torch.Tensor, scale: float,
                        kv_cache_dtype: str = "auto", k_scale: Optional[torch.Tensor] = None,
                        v_scale: Optional[torch.Tensor] = None, *, out_lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention of one query token a row over the row's selected pages: `paged_attention_decode` where row r
    and kv head h see only the tokens of `pages[r, h]` (int32 (rows, kv_heads, budget), numbers of the sequence's pages;
    negative entries and pages past the sequence are none) that lie below `seq_lens[r]`. A page listed twice counts
    twice. With nothing left a row answers zeros. `out_lse` (rows, q_heads) fp32 gets the natural-log sum-exp of the
    scaled scores (-inf for nothing), so that answers over disjoint pages can be merged (`merge_partials`). A NaN in a
    head's query or among its visible keys, or a logit past fp32's greatest, makes the head NaN; one below its lowest is
    -inf and has no weight. An fp8 cache's query may have any magnitude bf16 has: each head is scaled by a power of two."""
    qshape, qs = _query(query)
    os = out.stride()
    if out.shape != qshape or out.dtype is not query.dtype or os[2] != 1:
        raise ValueError(f"{_WHO}: out is {tuple(out.shape)} {out.dtype} strides {tuple(os)}; it must match query "
                         f"{tuple(qshape)} {query.dtype}")
    rows, hq, d = qshape
    (nb, page, hkv, cd), ks, vs = _cache_strides(key_cache, value_cache)
    width, stride = _tables(block_tables, seq_lens, rows)
    pshape, ps = pages.shape, pages.stride()
    if pages.dtype is not _I32 or len(pshape) != 3 or ps[2] != 1:
        _index("pages", pages, 3)
    listed, heads, budget = pshape
    if cd != d or listed != rows or heads != hkv:
        raise ValueError(f"{_WHO}: pages is {tuple(pages.shape)} beside query {tuple(qshape)} and key_cache "
                         f"{tuple(key_cache.shape)}; ({rows}, {hkv}, budget) and one head size needed")
    lse = 0
    if out_lse is not None:
        if out_lse.dtype is not _F32 or out_lse.shape != (rows, hq) or not out_lse.is_contiguous():
            raise ValueError(f"{_WHO}: out_lse is {tuple(out_lse.shape)} {out_lse.dtype}; contiguous ({rows}, {hq}) float32 needed")
        lse = out_lse.data_ptr()
    code = _code(kv_cache_dtype, key_cache, query.dtype)
    fp8 = code == _lib.KV_FP8_E4M3
    scale = _positive(scale)
    stream = _on(query, out, key_cache, value_cache, block_tables, seq_lens, pages, k_scale, v_scale, out_lse)
    rc = _lib.load().hkb_paged_sparse_decode(_lib.SPARSE_DECODE(
        out.data_ptr(), os[0], os[1], lse, query.data_ptr(), qs[0], qs[1],
        key_cache.data_ptr(), ks[0], ks[1], ks[2], nb, value_cache.data_ptr(), vs[0], vs[1], vs[2], nb,
        block_tables.data_ptr(), stride, width, seq_lens.data_ptr(), pages.data_ptr(), ps[0], ps[1], budget,
        rows, hq, hkv, d, page, code, _scale_ptr(k_scale, fp8, "k_scale") or 0, _scale_ptr(v_scale, fp8, "v_scale") or 0,
        scale), stream)
    if rc:
        _lib.check("hkb_paged_sparse_decode", rc)
    return out
