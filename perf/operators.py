"""Decode attention over a page selection, and the page bookkeeping under it: cases to measure.

Five operators of a serving step over a block-paged KV cache (`hk_dsl_b200.ops.paged_sparse`):

  tables  block tables, slot mapping and positions built on the GPU from request lengths
  bounds  per page, kv head and channel the least and the greatest key: a page's summary
  scores  for every query row, kv head and page the bound of its best logit, from the summary
  select  the budget's best pages of every row and kv head (ties go to the lowest page)
  attend  attention of one new token over the selected pages

`run` computes them in elementary torch operations, or makes the framework's calls where `own` is set.
Lengths are spread evenly over a case's range, so that `work` knows their sum; the seed orders them."""

import math

import torch

own = False

FIRST, LAST = 1, 4          # pages always kept: the sequence's first page and its newest four


# ----------------------------------------------------------------------------- cases

def _attn(op, batch, q_heads, kv_heads, lo, hi, dim=128, page=16, kv="bf16", budget=0, layout="heads"):
    return dict(op=op, batch=batch, q_heads=q_heads, kv_heads=kv_heads, lo=lo, hi=hi, dim=dim, page=page, kv=kv,
                budget=budget, layout=layout)


def _tables(batch, lo, hi, prompts, prompt, finished, page=16):
    return dict(op="tables", batch=batch, lo=lo, hi=hi, prompts=prompts, prompt=prompt, finished=finished, page=page)


def listed():
    return [
        # one decode step of the Llama-3-8B-shaped batch: every request gets one token
        dict(_tables(64, 2048, 8192, 0, 0, 0), name="tables, 64 decoding"),
        # a large mixed step: 2048 requests, 48 prompts of 2731 tokens come in, 64 requests shrink to an eighth
        dict(_tables(2048, 64, 4096, 48, 2731, 64), name="tables, 2048 mixed"),
        # the same decode step: each request's newest page is summarised again
        dict(_attn("bounds", 64, 32, 8, 2048, 8192), name="bounds, 64 decoding", new=1),
        # four prompts of 8192 tokens have just been written
        dict(_attn("bounds", 4, 32, 8, 8192, 8192, layout="tokens"), name="bounds, 4 x 8192 prompts", new=8192),
        # the small ragged batch
        dict(_attn("scores", 4, 8, 2, 64, 512), name="scores, 4 short"),
        # long context: two requests of 131072 tokens, eight query heads a kv head
        dict(_attn("scores", 2, 64, 8, 131072, 131072), name="scores, 2 x 131072"),
        # the Llama-3-8B-shaped batch, 1024 tokens kept
        dict(_attn("select", 64, 32, 8, 2048, 8192, budget=64), name="select, 64 of 128..512"),
        # long context, 4096 tokens kept
        dict(_attn("select", 2, 64, 8, 131072, 131072, budget=256), name="select, 256 of 8192"),
        # a single request with a budget of 37 pages: latency
        dict(_attn("attend", 1, 32, 8, 5000, 5000, budget=37), name="attend, 1 x 37 pages"),
        # the Llama-3-8B-shaped batch, 1024 tokens kept
        dict(_attn("attend", 64, 32, 8, 2048, 8192, budget=64), name="attend, 64 x 64 pages"),
        # the Qwen3-8B-shaped batch over an fp8 cache, 2048 tokens kept where a request has them
        dict(_attn("attend", 128, 32, 8, 1024, 4096, kv="fp8", budget=128), name="attend fp8, 128 x 128 pages"),
        # long context, 8192 tokens kept
        dict(_attn("attend", 2, 64, 8, 131072, 131072, budget=512), name="attend, 2 x 512 pages"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "bounds", "scores", "select", "attend"])
    if op == "tables":
        batch = _spread(rng, 1, 2048)
        prompts = rng.randint(0, batch // 4)
        finished = rng.randint(0, batch // 4)
        return _tables(batch, _spread(rng, 1, 64), _spread(rng, 64, 4096), prompts,
                       _spread(rng, 2, max(2, min(8192, 131072 // max(1, prompts)))), finished,
                       rng.choice([16, 16, 48, 64, 256]))
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice(["bf16", "fp16", "fp8"])
    page = rng.choice([16, 16, 32, 48, 64])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]) if kv_heads < 8 else rng.choice([1, 2, 4, 7, 8])
    batch = _spread(rng, 1, 128)
    # the cache's tokens are bounded: long sequences come in small batches
    hi = _spread(rng, 17, min(131072, 262144 // batch * 128 // dim))
    lo = hi if rng.random() < 0.3 else _spread(rng, 1, hi)
    case = _attn(op, batch, kv_heads * group, kv_heads, lo, hi, dim, page, kv, layout=rng.choice(["heads", "tokens"]))
    if op == "bounds":
        case["new"] = rng.choice([1, 1, _spread(rng, 1, lo)])
    if op == "select":              # there is something to leave out
        case["hi"] = max(hi, 2 * page * (FIRST + LAST))
        case["budget"] = min(_spread(rng, FIRST + LAST, 512), _ceil(case["hi"], page) - 3)
    if op == "attend":
        case["budget"] = _spread(rng, FIRST + LAST, 512)
        # no more bytes of selected tokens than the largest listed case reads
        per_page = batch * kv_heads * page * 2 * dim * (1 if kv == "fp8" else 2)
        case["budget"] = max(FIRST + LAST, min(case["budget"], 490_000_000 // per_page))
    return case


def _lens(case):
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _news(case):
    """A table step's new tokens a request: prompts come in, finished requests give back seven eighths, the others decode."""
    lens = _lens(case)
    new = [1] * case["batch"]
    for i in range(case["finished"]):
        new[i] = -(lens[i] * 7 // 8)
    for i in range(case["prompts"]):
        new[case["batch"] - 1 - i] = case["prompt"]
    return new


# ----------------------------------------------------------------------------- inputs

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}


def _rng(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)


def _page_table(pages, width, pool, gen):
    """A scrambled block table: request i owns pages[i] pages of the pool. Also the pages that nobody owns."""
    perm = torch.randperm(pool, generator=gen).to(torch.int32)
    n = torch.tensor(pages)
    start = torch.cumsum(n, 0) - n
    col = torch.arange(width)
    at = (start[:, None] + col).clamp(max=max(0, pool - 1))
    table = torch.where(col < n[:, None], perm[at], torch.zeros((), dtype=torch.int32))
    return table.cuda(), perm[sum(pages):]


def _normal(shape, kv, gen):
    """Standard normal values as the cache holds them; an fp8 cache keeps them over its scale, 5.6 / 448."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return (x / (5.6 / 448)).clamp(-448, 448).to(torch.float8_e4m3fn) if kv == "fp8" else x.to(_DTYPES[kv])


def _cache(case, blocks, gen):
    """(blocks, page, kv_heads, dim), stored heads first or tokens first."""
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    if case["layout"] == "heads":
        return _normal((blocks, h, p, d), case["kv"], gen).transpose(1, 2)
    return _normal((blocks, p, h, d), case["kv"], gen)


def prepare(case, seed):
    host, dev = _rng(seed)
    order = torch.randperm(case["batch"], generator=host).tolist()
    lens = [_lens(case)[i] for i in order]
    p = case["page"]
    s = dict(case=case, lens=torch.tensor(lens, dtype=torch.int32).cuda())
    if case["op"] == "tables":
        new = [_news(case)[i] for i in order]
        pages = [_ceil(n, p) for n in lens]
        after = [_ceil(max(0, n + k), p) for n, k in zip(lens, new)]
        width = max(max(pages), max(after)) + 1
        grow = sum(max(0, b - a) for a, b in zip(pages, after))
        pool = sum(pages) + grow + 64
        s["table"], spare = _page_table(pages, width, pool, host)
        s["free"] = torch.zeros(pool, dtype=torch.int32)
        s["free"][:spare.numel()] = spare
        s["free"] = s["free"].cuda()
        s["count"] = torch.tensor([spare.numel()], dtype=torch.int32).cuda()
        s["new"] = torch.tensor(new, dtype=torch.int32).cuda()
        s["back"] = -s["new"]
        tokens = max(1, sum(max(0, k) for k in new), sum(max(0, -k) for k in new))
        for side in ("there", "back_out"):
            s[side] = dict(slots=torch.zeros(tokens, dtype=torch.int64, device="cuda"),
                           positions=torch.zeros(tokens, dtype=torch.int64, device="cuda"),
                           start=torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda"),
                           status=torch.zeros(case["batch"], dtype=torch.int32, device="cuda"))
        return s
    pages = [_ceil(n, p) for n in lens]
    width, blocks = max(pages), sum(pages) + 3
    h, d, hq, rows = case["kv_heads"], case["dim"], case["q_heads"], case["batch"]
    act = torch.float16 if case["kv"] == "fp16" else torch.bfloat16
    s["scale"] = d ** -0.5
    s["kv"] = "fp8" if case["kv"] == "fp8" else "auto"
    s["k_scale"] = torch.tensor([5.6 / 448]).cuda() if case["kv"] == "fp8" else None
    s["v_scale"] = torch.tensor([5.6 / 448]).cuda() if case["kv"] == "fp8" else None
    s["table"], _ = _page_table(pages, width, blocks, host)
    if case["op"] in ("bounds", "attend"):
        s["k"] = _cache(case, blocks, dev)
    if case["op"] == "bounds":
        new = case["new"]
        s["start"] = (torch.arange(rows + 1, dtype=torch.int32) * new).cuda()
        s["tokens"] = rows * new
        s["touched"] = sum(_ceil(n, p) - (n - new) // p for n in lens)
        s["bounds"] = _normal((blocks, h, 2, d), case["kv"], dev)
    if case["op"] == "scores":
        s["bounds"] = torch.empty((blocks, h, 2, d), device="cuda", dtype=_DTYPES[case["kv"]])
        for a in range(0, blocks, 4096):
            x = _normal((min(4096, blocks - a), h, p, d), case["kv"], dev).float()
            s["bounds"][a:a + 4096] = torch.stack((x.amin(2), x.amax(2)), 2).to(s["bounds"].dtype)
        s["q"] = torch.randn((rows, hq, d), generator=dev, device="cuda").to(act)
        s["scores"] = torch.empty((rows, h, width), device="cuda")
    if case["op"] == "select":
        x = torch.randn((rows, h, width), generator=dev, device="cuda") * 2 + 18
        dead = torch.arange(width, device="cuda") >= torch.tensor(pages, device="cuda")[:, None, None]
        s["scores"] = x.masked_fill(dead, -math.inf)
        s["pages"] = torch.empty((rows, h, case["budget"]), dtype=torch.int32, device="cuda")
    if case["op"] == "attend":
        s["v"] = _cache(case, blocks, dev)
        s["q"] = torch.randn((rows, hq, d), generator=dev, device="cuda").to(act)
        # a selection as it comes: random pages, the first and the newest among them, ascending, -1 behind
        n = torch.tensor(pages, device="cuda")[:, None, None]
        col = torch.arange(width, device="cuda")
        key = torch.rand((rows, h, width), generator=dev, device="cuda") + 2 * ((col < FIRST) | (col >= n - LAST))
        key = key.masked_fill(col >= n, -1.0)
        k = min(width, case["budget"])
        best = torch.topk(key, k).indices
        best = torch.where(torch.arange(k, device="cuda") < n, best, width).sort(-1).values
        s["pages"] = torch.full((rows, h, case["budget"]), -1, dtype=torch.int32, device="cuda")
        s["pages"][:, :, :k] = torch.where(best < width, best, -1).to(torch.int32)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((rows, hq), device="cuda")
    return s


# ----------------------------------------------------------------------------- the operators, plainly

def _advance(table, lens, new, free, count, out, page):
    """Grow (new > 0) or shrink requests, in place; pages come from and go to the stack free[:count]."""
    width, tokens = table.shape[1], out["slots"].numel()
    dev = table.device
    old, new = lens.clamp(min=0).long(), new.long()
    after, query = (old + new).clamp(min=0), new.clamp(min=0)
    ends = query.cumsum(0)
    start = ends - query
    have = ((old + page - 1) // page).clamp(max=width)
    want = (after + page - 1) // page
    grows = new > 0
    status = torch.where(grows & (want > width), 2, torch.where(grows & (ends > tokens), 3, 0))
    need = torch.where((status == 0) & grows, (want - have).clamp(min=0), 0)
    upto = need.cumsum(0)
    status = torch.where((need > 0) & (upto > count), 1, status)
    ok = status == 0
    first = upto - need                              # a request's pages come from the stack's top downwards
    take = torch.where(ok, need, 0)
    give = torch.where(new < 0, (have - want).clamp(min=0), 0)
    given = give.cumsum(0)

    def page_of(r, logical):
        fresh = free[(count - 1 - (first[r] + logical - have[r])).clamp(0, free.numel() - 1)]
        return torch.where(logical < have[r], table[r, logical.clamp(0, width - 1)], fresh).long()

    t = torch.arange(tokens, device=dev)
    r = torch.searchsorted(ends, t, right=True)
    real = r < lens.numel()
    r = r.clamp(max=lens.numel() - 1)
    pos = old[r] + t - start[r]
    block = page_of(r, pos // page)
    out["slots"].copy_(torch.where(real & ok[r] & (block >= 0), block * page + pos % page, -1))
    out["positions"].copy_(torch.where(real, pos, 0))
    out["start"][1:].copy_(ends)
    out["status"].copy_(status)

    col = torch.arange(width, device=dev)
    every = torch.arange(lens.numel(), device=dev)[:, None]
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    grown = torch.where(fresh, page_of(every, col[None, :]).int(), table)
    left = count - take.sum()
    at = torch.arange(free.numel(), device=dev) - left
    giver = torch.searchsorted(given, at.clamp(min=0), right=True)
    back = (at >= 0) & (giver < lens.numel())
    giver = giver.clamp(max=lens.numel() - 1)
    which = (want[giver] + at - (given - give)[giver]).clamp(0, width - 1)
    free.copy_(torch.where(back, table[giver, which], free))
    table.copy_(grown)
    lens.copy_(torch.where(ok, after, old))
    count.copy_((left + given[-1:]).clamp(max=free.numel()))


def _bounds(s):
    """The channelwise least and greatest key of every page that holds one of the last new tokens."""
    c, k, p, lens = s["case"], s["k"], s["case"]["page"], s["lens"].long()
    new = (s["start"][1:] - s["start"][:-1]).long()
    first, last = (lens - new) // p, (lens + p - 1) // p
    count = last - first
    r = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), count, output_size=s["touched"])
    logical = first[r] + torch.arange(s["touched"], device="cuda") - (count.cumsum(0) - count)[r]
    block = s["table"][r, logical].long()
    live = (logical[:, None] * p + torch.arange(p, device="cuda") < lens[r][:, None])[:, :, None, None]
    x = k[block].float()
    s["bounds"][block] = torch.stack((torch.where(live, x, math.inf).amin(1), torch.where(live, x, -math.inf).amax(1)),
                                     2).to(k.dtype)
    return s["bounds"].float() if c["kv"] == "fp8" else s["bounds"]


def _unit(s, name):
    return s[name] if s[name] is not None else 1.0


def _scores(s):
    """max over the group's heads of sum_d max(q_d low_d, q_d high_d): positive parts meet the upper bounds, negative the lower."""
    c = s["case"]
    b = s["bounds"][s["table"].long()].float()
    q = s["q"].float().view(c["batch"], c["kv_heads"], -1, c["dim"])
    low, high = b[:, :, :, 0].permute(0, 2, 3, 1), b[:, :, :, 1].permute(0, 2, 3, 1)
    x = (q.clamp(min=0) @ high + q.clamp(max=0) @ low).amax(2) * (s["scale"] * _unit(s, "k_scale"))
    pages = (s["lens"] + c["page"] - 1) // c["page"]
    return x.masked_fill(torch.arange(x.shape[2], device="cuda") >= pages[:, None, None], -math.inf)


def _select(s):
    """The budget's greatest scores, first and newest pages before all, ties to the lowest page; ascending, -1 behind."""
    c, x = s["case"], s["scores"] + 0.0
    col = torch.arange(x.shape[2], device="cuda")
    pages = ((s["lens"] + c["page"] - 1) // c["page"])[:, None, None]
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
    key = torch.where(torch.isnan(x), 1 << 33, key)
    key = torch.where((col < FIRST) | (col >= pages - LAST), 1 << 34, key)
    key = torch.where(col >= pages, -(1 << 34), key)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :, :c["budget"]]
    best = torch.where(torch.arange(best.shape[2], device="cuda") < pages, best, x.shape[2]).sort(-1).values
    best = torch.where(best < x.shape[2], best, -1)
    return torch.nn.functional.pad(best, (0, c["budget"] - best.shape[2]), value=-1).to(torch.int32)


def _attend(s):
    c, pages = s["case"], s["pages"].long()
    rows, h, k = pages.shape
    row, head = torch.arange(rows, device="cuda")[:, None, None], torch.arange(h, device="cuda")[None, :, None]
    block = s["table"][row, pages.clamp(min=0)].long()
    token = pages[..., None] * c["page"] + torch.arange(c["page"], device="cuda")
    live = ((pages[..., None] >= 0) & (token < s["lens"][:, None, None, None])).view(rows, h, 1, -1)
    keys = s["k"][block, :, head].float().view(rows, h, -1, c["dim"])
    q = s["q"].float().view(rows, h, -1, c["dim"])
    x = (q @ keys.transpose(2, 3)) * (s["scale"] * _unit(s, "k_scale"))
    x = torch.where(live, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(-1, keepdim=True)
    values = s["v"][block, :, head].float().view(rows, h, -1, c["dim"])
    values = torch.where(live.view(rows, h, -1, 1), values, 0.0)
    o = (w @ values) * (_unit(s, "v_scale") / torch.where(total > 0, total, 1.0))
    return o.view(rows, -1, c["dim"]).to(s["q"].dtype), (top + torch.log(total)).view(rows, -1)


# ----------------------------------------------------------------------------- one pass

def _tables_out(s):
    return {"table": s["table"], "lens": s["lens"], "free": s["free"], "count": s["count"], **s["there"],
            "back": s["back_out"]}


def run(s):
    c = s["case"]
    if own:
        from hk_dsl_b200.ops import paged_sparse as ps
        if c["op"] == "tables":
            for new, o in ((s["new"], s["there"]), (s["back"], s["back_out"])):
                ps.advance_tables(s["table"], s["lens"], new, s["free"], s["count"], c["page"], o["slots"],
                                  o["positions"], o["start"], o["status"])
            return _tables_out(s)
        if c["op"] == "bounds":
            if c["new"] == 1:
                ps.update_page_bounds(s["bounds"], s["k"], s["table"], s["lens"])
            else:
                ps.update_page_bounds(s["bounds"], s["k"], s["table"], s["lens"], s["start"], num_tokens=s["tokens"])
            return s["bounds"].float() if c["kv"] == "fp8" else s["bounds"]
        if c["op"] == "scores":
            return ps.page_scores(s["scores"], s["q"], s["bounds"], s["table"], s["lens"], s["scale"], c["page"],
                                  s["kv"], s["k_scale"])
        if c["op"] == "select":
            return ps.select_pages(s["pages"], s["scores"], s["lens"], c["page"], first=FIRST, last=LAST)
        ps.paged_sparse_decode(s["out"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["pages"], s["scale"], s["kv"],
                               s["k_scale"], s["v_scale"], out_lse=s["lse"])
        return s["out"], s["lse"]
    if c["op"] == "tables":
        # a step, and its taking back (rejected drafts, a request that makes room for the next of its size)
        _advance(s["table"], s["lens"], s["new"], s["free"], s["count"], s["there"], c["page"])
        _advance(s["table"], s["lens"], s["back"], s["free"], s["count"], s["back_out"], c["page"])
        return _tables_out(s)
    return {"bounds": _bounds, "scores": _scores, "select": _select, "attend": _attend}[c["op"]](s)


# ----------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    lens, p = _lens(case), case["page"]
    pages = [_ceil(n, p) for n in lens]
    if case["op"] == "tables":
        new = _news(case)
        moved = sum(abs(_ceil(max(0, n + k), p) - _ceil(n, p)) for n, k in zip(lens, new))
        tokens = 2 * max(1, sum(max(0, k) for k in new), sum(max(0, -k) for k in new))
        # two calls: lengths in and out, new tokens, starts, status; a slot and a position a token; a page read and written
        return {"bytes": 2 * 20 * case["batch"] + 16 * tokens + 2 * 8 * moved, "flops": 0}
    h, d, hq, rows = case["kv_heads"], case["dim"], case["q_heads"], case["batch"]
    es = 1 if case["kv"] == "fp8" else 2
    if case["op"] == "bounds":
        new = case["new"]
        read = sum(n - (n - new) // p * p for n in lens)
        touched = sum(_ceil(n, p) - (n - new) // p for n in lens)
        return {"bytes": (read + 2 * touched) * h * d * es + 4 * touched, "flops": 2 * read * h * d}
    if case["op"] == "scores":
        n = sum(pages)
        return {"bytes": n * (h * 2 * d * es + 4) + rows * hq * d * 2 + 4 * rows * h * max(pages), "flops": 4 * n * hq * d}
    if case["op"] == "select":
        return {"bytes": 4 * h * (sum(pages) + rows * case["budget"]), "flops": h * sum(pages)}
    # the newest page is always selected: what it lacks to a whole page is not read
    tokens = sum(min(n, k * p) - (0 if n <= k * p else -n % p) for n, k in zip(lens, [case["budget"]] * rows))
    return {"bytes": h * tokens * 2 * d * es + 2 * rows * hq * d * 2 + 4 * rows * (hq + h * case["budget"]),
            "flops": 4 * tokens * hq * d}


# ----------------------------------------------------------------------------- in 64 bits, from the definitions

def exact(case, seed):
    if case["op"] in ("tables", "select"):
        return None                      # whole numbers
    s = prepare(case, seed)
    lens, table, p, h, d = s["lens"].tolist(), s["table"].long(), case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "bounds":
        want = s["bounds"].double()
        for i, n in enumerate(lens):
            for j in range((n - case["new"]) // p, _ceil(n, p)):
                rows = s["k"][table[i, j], :min(p, n - j * p)].double()
                want[table[i, j], :, 0], want[table[i, j], :, 1] = rows.min(0).values, rows.max(0).values
        return want
    q = s["q"].double()
    group = case["q_heads"] // h
    if case["op"] == "scores":
        want = torch.full(s["scores"].shape, -math.inf, dtype=torch.float64, device="cuda")
        unit = float(s["k_scale"]) if case["kv"] == "fp8" else 1.0
        for i, n in enumerate(lens):
            for a in range(0, _ceil(n, p), 512):
                ids = table[i, a:min(a + 512, _ceil(n, p))]
                lo, hi = s["bounds"][ids].double().unbind(2)               # (pages, kv heads, dim)
                lo, hi = (b.repeat_interleave(group, 1) for b in (lo, hi))
                best = torch.maximum(q[i] * lo, q[i] * hi).sum(-1).view(-1, h, group).amax(-1)
                want[i, :, a:a + ids.numel()] = best.T * s["scale"] * unit
        return want
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    ks, vs = (float(s["k_scale"]), float(s["v_scale"])) if case["kv"] == "fp8" else (1.0, 1.0)
    chosen = s["pages"].tolist()
    for i, n in enumerate(lens):
        for g in range(h):
            mine = torch.tensor([j for j in chosen[i][g] if j >= 0], device="cuda")
            at = (mine[:, None] * p + torch.arange(p, device="cuda")).flatten()
            at = at[at < n]
            ids = table[i][at // p]
            heads = slice(g * group, (g + 1) * group)
            x = q[i, heads] @ s["k"][ids, at % p, g].double().T * (s["scale"] * ks)
            lse[i, heads] = torch.logsumexp(x, -1)
            out[i, heads] = torch.softmax(x, -1) @ s["v"][ids, at % p, g].double() * vs
    return out, lse
