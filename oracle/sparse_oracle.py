"""CPU oracle of decode over selected pages and the page bookkeeping under it. TEST INFRASTRUCTURE ONLY.

Each operator from its definition, one request, row and head at a time, in Python integers and float64. Nothing of
the product is used here. The bounds `*_tol` say how far a kernel may be off, counted from its roundings:
u = half a step of a type, relative to the value (bf16 2^-8, fp16 2^-11, fp32 2^-24).
"""

from __future__ import annotations

import math

import torch

U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
OK, NO_PAGES, TABLE_FULL, NO_ROWS = 0, 1, 2, 3


def ceil_div(a: int, b: int) -> int:
    return -(-a // b)


def as_float64(c: torch.Tensor, scale=None) -> torch.Tensor:
    if c.dtype == torch.uint8:
        c = c.view(torch.float8_e4m3fn)
    x = c.float().double()
    return x if scale is None else x * float(scale)


# ------------------------------------------------------------------------- tables

def advance_ref(table, lens, new, free, count, page, rows):
    """All lists of Python integers (`table` a list of lists), nothing in place:
    (table, lens, free, count, slots, positions, starts, status)."""
    table, lens, free = [list(r) for r in table], list(lens), list(free)
    width, cap = len(table[0]) if table else 0, len(free)
    count = max(0, min(count, cap))
    stack, used, short = free[:count], 0, False
    starts, status, slots, positions, back = [0], [], [-1] * rows, [0] * rows, []
    for i, n in enumerate(new[:len(lens)]):
        old = max(0, lens[i])
        after, have = max(0, old + n), min(ceil_div(old, page), width)
        t0 = starts[-1]
        starts.append(t0 + max(0, n))
        st = OK
        if n > 0:
            want = ceil_div(after, page)
            if want > width or after > 2 ** 31 - 1:
                st = TABLE_FULL
            elif starts[-1] > rows:
                st = NO_ROWS
            elif want > have:
                # the sum of what was asked for runs on past a request that did not get it
                used += want - have
                if used > count:
                    st = NO_PAGES
                else:
                    for k in range(want - have):
                        table[i][have + k] = stack[count - 1 - (used - (want - have) + k)]
        elif n < 0:
            want = ceil_div(after, page)
            back += table[i][want:have]
        for j in range(min(max(0, n), max(0, rows - t0))):
            if t0 + j < rows:
                pos = old + j
                block = table[i][pos // page] if st == OK else -1
                slots[t0 + j] = block * page + pos % page if block >= 0 else -1
                positions[t0 + j] = pos
        lens[i] = after if st == OK else old
        status.append(st)
    # pages handed out: the stack's top ones
    taken = 0
    for i, n in enumerate(new[:len(lens)]):
        if n > 0 and status[i] == OK:
            old = lens[i] - n
            taken += max(0, ceil_div(lens[i], page) - min(ceil_div(old, page), width))
    left = count - taken
    for k, p in enumerate(back):
        if left + k < cap:
            free[left + k] = p
    return table, lens, free, min(cap, left + len(back)), slots, positions, starts, status


# ------------------------------------------------------------------------- bounds

def bounds_ref(bounds, key_cache, table, lens, starts=None):
    """The summary tensor after the call (a copy): exact, values of the cache's type."""
    out = bounds.clone()
    raw = key_cache.dtype == torch.uint8
    page = key_cache.shape[1]
    for i, n in enumerate(lens):
        new = 1 if starts is None else max(1, starts[i + 1] - starts[i])
        if n <= 0:
            continue
        for j in range(max(0, n - new) // page, ceil_div(n, page)):
            if j >= table.shape[1]:
                break
            b = int(table[i, j])
            if not 0 <= b < min(out.shape[0], key_cache.shape[0]):
                continue
            rows = as_float64(key_cache[b, :min(page, n - j * page)])
            for which, x in ((0, rows.amin(0)), (1, rows.amax(0))):
                x = x.float().to(torch.float8_e4m3fn if raw else key_cache.dtype)
                out[b, :, which] = x.view(torch.uint8) if raw else x
    return out


# ------------------------------------------------------------------------- scores

def scores_ref(q, bounds, table, lens, page, scale, k_scale=None):
    """(scores float64, tolerance float64): the bound of a page's logits from its summary, -inf behind the sequence.
    The kernel multiplies exact products of 16-bit values and adds 2 D of them in fp32, each addition off by at most
    2^-23 (the tensor core may cut) of the sum of magnitudes; then three roundings of the result. An fp8 cache's query is
    rounded to fp16 after scaling by a power of two: 2^-38 of its largest value at most."""
    rows, hq, d = q.shape
    hkv = bounds.shape[1]
    g = hq // hkv
    out = torch.full((rows, hkv, table.shape[1]), -math.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    b64, q64 = as_float64(bounds), q.double()
    unit = scale * (1.0 if k_scale is None else float(k_scale))
    for r in range(rows):
        for p in range(min(ceil_div(max(0, lens[r]), page), table.shape[1])):
            lo, hi = b64[int(table[r, p].clamp(0, bounds.shape[0] - 1))].unbind(1)     # (kv heads, D)
            for h in range(hkv):
                qq = q64[r, h * g:(h + 1) * g]
                out[r, h, p] = torch.maximum(qq * lo[h], qq * hi[h]).sum(-1).amax() * unit
                # an infinite bound is no part of a finite score, and so of none of its sums
                al, ah = (torch.where(torch.isinf(x[h]), 0.0, x[h].abs()) for x in (lo, hi))
                mag = (qq.abs() * torch.maximum(al, ah)).sum(-1).amax()
                small = 2.0 ** -38 * qq.abs().amax() * (al + ah).sum() if k_scale is not None else 0.0
                tol[r, h, p] = unit * (mag * (2 * d + 4) * 2.0 ** -23 + small)
    return out, tol


# ------------------------------------------------------------------------- selection

def select_ref(scores, lens, page, budget, first, last):
    rows, hkv, width = scores.shape
    out = torch.full((rows, hkv, budget), -1, dtype=torch.int32)
    for r in range(rows):
        n = min(ceil_div(max(0, lens[r]), page), width)
        for h in range(hkv):
            x = scores[r, h].tolist()

            def rank(p):
                if p < first or p >= n - last:
                    return (0, 0.0, p)
                return (1, 0.0, p) if math.isnan(x[p]) else (2, -x[p], p)

            best = sorted(sorted(range(n), key=rank)[:budget])
            out[r, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


# ------------------------------------------------------------------------- attention

def sparse_ref(q, key_cache, value_cache, table, lens, pages, scale, k_scale=None, v_scale=None, terms=1):
    """(out, out tolerance, lse, lse tolerance), float64. What the kernel rounds: q.k is exact products added in fp32
    (2^-23 of the sum of magnitudes an addition), the exponential's argument and the exponential (2^-21 together), the
    weights to 16 bits before they meet V -- the activation type's u, fp16's for an fp8 cache, plus fp16's smallest
    step under values of 1 and more -- and the answer to the activation type. `terms` 2: a weight is its upper half and,
    below 2^-7 of it, the rest rounded to bf16."""
    rows, hq, d = q.shape
    page, hkv = key_cache.shape[1], key_cache.shape[2]
    g = hq // hkv
    fp8 = key_cache.dtype not in U16
    up = 2.0 ** -11 if fp8 else U16[q.dtype] if terms == 1 else 2.0 ** -7 * U16[torch.bfloat16]
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    for r in range(rows):
        n = max(0, lens[r])
        for h in range(hkv):
            at = [j * page + t for j in pages[r, h].tolist() if 0 <= j < table.shape[1] for t in range(page) if j * page + t < n]
            if not at:
                continue
            ids = torch.tensor([int(table[r, t // page].clamp(0, key_cache.shape[0] - 1)) for t in at])
            off = torch.tensor([t % page for t in at])
            kk = as_float64(key_cache[ids, off, h], k_scale)
            vv = as_float64(value_cache[ids, off, h], v_scale)
            for hh in range(h * g, (h + 1) * g):
                qq = q[r, hh].double()
                x = kk @ qq * scale
                lse[r, hh] = torch.logsumexp(x, 0)
                w = torch.softmax(x, 0)
                out[r, hh] = w @ vv
                ds = float((kk.abs() @ qq.abs()).amax() * scale) * (d + 4) * 2.0 ** -23 + float(x.abs().amax()) * 2.0 ** -23 + 2.0 ** -21
                a = w @ vv.abs()
                sub = len(at) * 2.0 ** -25 * vv.abs().amax() if q.dtype == torch.float16 or fp8 else 0.0
                tol[r, hh] = out[r, hh].abs() * U16[q.dtype] + a * (up + 3 * ds + 2.0 ** -18) + sub
                lse_tol[r, hh] = 2 * ds + (abs(float(lse[r, hh])) + 1) * 2.0 ** -22
    return out, tol, lse, lse_tol
