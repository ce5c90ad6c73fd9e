"""Serving operators of Selective Attention: what a program that answers many requests at once has them do, as cases that can be
timed and compared.

Four operators over one paged cache.  Requests (rows) own pages of ``page_size`` tokens; K and V of a layer are pools of pages,
(pages, H, page_size, D), and each row has its history sums, ``selected`` (rows, G, capacity).

    tables    ``paged.append_tokens``: from the number of new tokens of every row, the pages that the rows get, their block
              tables, and the slot of every new token
    attend    ``paged.paged_attention``: the new tokens (packed, row after row: a prompt, a further chunk of one, a single
              token) go into the pages and attend to all of their row's tokens under Selective Attention; the history moves on
    select    ``beams.beam_select``: the best continuations over beams and vocabulary
    reorder   ``paged.reorder_rows`` and ``paged.move_rows``: every beam becomes a copy of its parent; full pages are shared,
              the page that is still being filled and the history are copied

``run`` has each in its plain form, or (``own``) by the framework's calls.
"""

import math
import os
import random
import sys

import torch

own = False
PACKAGE = os.path.join(os.getcwd(), "selective-attention-study_b200")


def _framework():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from selective_attention_b200 import beams, paged

    return paged, beams


# ---- cases --------------------------------------------------------------------------------------------------------------------

def _tables(name=None, *, rows, page, ragged, prompts, tokens, decoding):
    """``prompts`` of the rows get about ``tokens`` new tokens each, the others one; ``decoding``: about how many tokens a row has."""
    c = dict(kind="tables", rows=rows, page=page, ragged=ragged, prompts=prompts, tokens=tokens, decoding=decoding)
    return c if name is None else dict(c, name=name)


def _attend(name=None, *, rows, heads, dim, page, ragged, prompts, tokens, cached, per_head=False, exempt=1, scale=0.3):
    """``prompts`` of the rows get about ``tokens`` new tokens, the others one, after about ``cached`` (exactly: one row);
    ``scale``: of q and k, which sets how fast the history grows."""
    c = dict(kind="attend", rows=rows, heads=heads, dim=dim, page=page, ragged=ragged, prompts=prompts, tokens=tokens, cached=cached,
             per_head=per_head, exempt=exempt, scale=scale)
    return c if name is None else dict(c, name=name)


def _select(name=None, *, groups, beams, width, vocab, dtype):
    c = dict(kind="select", groups=groups, beams=beams, width=width, vocab=vocab, dtype=dtype)
    return c if name is None else dict(c, name=name)


def _reorder(name=None, *, groups, beams, heads, dim, page, tokens, ragged, per_head=False):
    c = dict(kind="reorder", groups=groups, beams=beams, heads=heads, dim=dim, page=page, tokens=tokens, ragged=ragged, per_head=per_head)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a decode step of 64 requests: one token each, a page now and then; latency
        _tables("tables-64-decoding", rows=64, page=16, ragged=1, prompts=0, tokens=1, decoding=4000),
        # a busy server takes in 120 long prompts while 392 rows decode: a quarter of a million slots
        _tables("tables-512-mixed", rows=512, page=16, ragged=2, prompts=120, tokens=2200, decoding=3000),
        # a chat-sized prompt of the 12-head model, alone: latency
        _attend("prompt-300", rows=1, heads=12, dim=64, page=16, ragged=0, prompts=1, tokens=300, cached=0),
        # a further chunk of a long prompt of the 16-head model
        _attend("chunk-2k-after-30k", rows=1, heads=16, dim=64, page=64, ragged=0, prompts=1, tokens=2048, cached=30000),
        # one step of a server: eight prompts in chunks and sixteen rows that decode, lengths as they come
        _attend("mixed-24-rows", rows=24, heads=16, dim=64, page=32, ragged=3, prompts=8, tokens=500, cached=3000),
        # head_dim 128, every head its own selector, four ragged chunks, the first 16 positions exempt
        _attend("chunks-d128-per-head", rows=4, heads=8, dim=128, page=128, ragged=4, prompts=4, tokens=1000, cached=2500, per_head=True,
                exempt=16),
        # one token after the long prompt of the benchmark
        _attend("decode-131k", rows=1, heads=16, dim=64, page=128, ragged=0, prompts=0, tokens=1, cached=131000, scale=1.0),
        # one token for each of 64 rows of very different lengths
        _attend("decode-64-ragged", rows=64, heads=16, dim=64, page=16, ragged=5, prompts=0, tokens=1, cached=3500),
        # four beams of one request over the decoder's vocabulary
        _select("select-4-beams", groups=1, beams=4, width=4, vocab=50304, dtype="fp32"),
        # eight beams of 32 requests, logits as the output projection leaves them
        _select("select-32x8-beams", groups=32, beams=8, width=8, vocab=50304, dtype="bf16"),
        # four beams of one request after a short prompt
        _reorder("reorder-4-beams", groups=1, beams=4, heads=12, dim=64, page=16, tokens=400, ragged=0),
        # eight beams of 32 requests, every head with a history of its own
        _reorder("reorder-32x8-per-head", groups=32, beams=8, heads=16, dim=64, page=64, tokens=1500, ragged=6, per_head=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tables", "attend", "attend", "decode", "decode", "select", "reorder"])
    ragged = rng.randint(10, 10**6)
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        rows = _log(rng, 1, 512)
        prompts = rng.randint(0, min(rows, 120))
        return _tables(rows=rows, page=page, ragged=ragged, prompts=prompts, tokens=_log(rng, 2, 2200), decoding=_log(rng, 1, 4000))
    if kind == "select":
        beams = rng.randint(1, 16)
        return _select(groups=_log(rng, 1, max(1, 256 // beams)), beams=beams, width=rng.randint(1, min(32, 2 * beams + 1)),
                       vocab=_log(rng, 200, 50304), dtype=rng.choice(["fp32", "bf16", "fp16"]))
    dim = rng.choice([64, 64, 128])
    heads = rng.choice([2, 3, 5, 8, 12, 16]) if dim == 64 else rng.choice([2, 3, 8])
    if kind == "reorder":
        beams = rng.randint(1, 12)
        return _reorder(groups=_log(rng, 1, max(1, 256 // beams)), beams=beams, heads=heads, dim=dim, page=page,
                        tokens=_log(rng, 1, 1500), ragged=ragged, per_head=rng.random() < 0.3)
    per_head, exempt, scale = rng.random() < 0.3, rng.choice([1, 1, 1, 16]), rng.choice([1.0, 0.3, 0.3, 0.1])
    if kind == "decode":
        rows = _log(rng, 1, 64)
        return _attend(rows=rows, heads=heads, dim=dim, page=page, ragged=ragged, prompts=0, tokens=1,
                       cached=_log(rng, 1, 131000 if rows == 1 else max(2, 220000 // rows)), per_head=per_head, exempt=exempt, scale=scale)
    rows = _log(rng, 1, 24)
    tokens = _log(rng, 2, 2048 if rows == 1 else 500)
    cached = 0 if rng.random() < 0.2 else _log(rng, 1, 30000 if rows == 1 else max(2, 72000 // rows))
    return _attend(rows=rows, heads=heads, dim=dim, page=page, ragged=ragged, prompts=rng.randint(1, rows), tokens=tokens, cached=cached,
                   per_head=per_head, exempt=exempt, scale=scale)


def _lengths(c):
    """(tokens that each row has, new tokens of each row), whole numbers that the case alone decides."""
    rng, rows = random.Random(c["ragged"]), c["rows"]
    about = c["decoding"] if c["kind"] == "tables" else c["cached"]
    if rows == 1:
        return [about], [c["tokens"] if c["prompts"] else 1]
    cached = [0 if about == 0 else rng.randint(1, 2 * about) for _ in range(rows)]
    counts = [rng.randint(2, 2 * c["tokens"]) if r < c["prompts"] else 1 for r in range(rows)]
    both = list(zip(cached, counts))
    rng.shuffle(both)                                          # rows that decode and rows with a prompt stand anyhow
    return [x for x, _ in both], [y for _, y in both]


# ---- the state that a program has in hand ------------------------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _normal(gen, shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _page_tables(rows, num_pages, page, max_pages, lengths, gen, heads):
    """Tables in which row r has the pages of ``lengths[r]`` tokens, taken from a pool in no order; one storage, so that one copy
    brings a saved state of them back."""
    sizes = {"block_tables": rows * max_pages, "lengths": rows, "free_pages": num_pages, "free_count": 1, "page_refs": num_pages}
    storage = torch.zeros(sum(sizes.values()), dtype=torch.int32, device="cuda")
    t = dict(zip(sizes, storage.split(list(sizes.values()))))
    t["block_tables"] = t["block_tables"].view(rows, max_pages)
    order = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    held = [-(-n // page) for n in lengths]
    row = torch.repeat_interleave(torch.arange(rows), torch.tensor(held))
    block = torch.cat([torch.arange(n) for n in held])
    n_held = sum(held)
    t["block_tables"].fill_(-1)
    t["block_tables"][row.cuda(), block.cuda()] = order[:n_held]
    t["page_refs"][order[:n_held].long()] = 1
    t["free_pages"][: num_pages - n_held] = order[n_held:]
    t["free_count"].fill_(num_pages - n_held)
    t["lengths"].copy_(_int32(lengths))
    return dict(t, page_size=page, heads=heads), storage


def _history(c, lengths, rows, groups, capacity, gen):
    """``selected``: what the tokens of each row have received by now: more the longer ago they were written, never negative, none
    for the exempt ones.  Behind a row's tokens stands what an earlier request left there."""
    age = (_int32(lengths)[:, None] - 1 - torch.arange(capacity, device="cuda")).clamp_min(0).float()[:, None]
    noise = torch.randn(rows, groups, capacity, generator=gen, device="cuda")
    selected = (0.4 * c.get("scale", 0.3) ** 2 * (age + noise * age.sqrt())).clamp_min(0.0) + noise.abs() * (age == 0)
    selected[:, :, : c.get("exempt", 1)] = 0.0
    return selected


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda").manual_seed(seed)
    if c["kind"] == "select":
        shape = (c["groups"], c["beams"], c["vocab"])
        logits = _normal(gen, shape, 2.5, DTYPES[c["dtype"]])
        scores = -torch.rand(shape[:2], generator=gen, device="cuda") * 8.0
        return {"case": c, "logits": logits, "scores": scores}
    if c["kind"] == "reorder":
        rows, page, h, d = c["groups"] * c["beams"], c["page"], c["heads"], c["dim"]
        groups, rng = (h if c["per_head"] else 1), random.Random(c["ragged"])
        tokens = [c["tokens"] if c["groups"] == 1 else rng.randint(1, 2 * c["tokens"]) for _ in range(c["groups"])]
        lengths = [n for n in tokens for _ in range(c["beams"])]
        max_pages = -(-max(lengths) // page) + 4
        num_pages = sum(-(-n // page) for n in lengths) + 3 * rows + 7
        tables, storage = _page_tables(rows, num_pages, page, max_pages, lengths, gen, h)
        # parents as beam search leaves them: most children come from a few good beams of their own request
        best = torch.randint(0, c["beams"], (c["groups"], c["beams"]), generator=gen, device="cuda")
        best = torch.minimum(best, torch.randint(0, c["beams"], best.shape, generator=gen, device="cuda"))
        parents = (best + torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]).to(torch.int32).reshape(-1)
        cache = {"k": _normal(gen, (num_pages, h, page, d)), "v": _normal(gen, (num_pages, h, page, d)),
                 "selected": _history(c, lengths, rows, groups, max_pages * page, gen)}
        return {"case": c, "tables": tables, "storage": storage, "saved": storage.clone(), "cache": cache,
                "history": cache["selected"].clone(), "parents": parents}
    cached, counts = _lengths(c)
    rows, page, heads = c["rows"], c["page"], c.get("heads", 16)
    after = [a + b for a, b in zip(cached, counts)]
    max_pages = -(-max(after) // page)
    num_pages = sum(-(-n // page) for n in after) + 5
    tables, storage = _page_tables(rows, num_pages, page, max_pages, cached, gen, heads)
    state = {"case": c, "tables": tables, "storage": storage, "saved": storage.clone(), "counts": _int32(counts), "total": sum(counts),
             "longest": max(after), "most": max(counts)}
    if c["kind"] == "tables":
        return state
    # the step's plan is made once and serves every layer
    h, d = heads, c["dim"]
    groups = h if c["per_head"] else 1
    if own:
        step = _framework()[0].append_tokens(tables, state["counts"], state["total"], max_length=state["longest"],
                                                max_count=state["most"])
    else:
        step = _plain_append(tables, state["counts"], state["total"])
    cache = {"k": _normal(gen, (num_pages, h, page, d), c["scale"]), "v": _normal(gen, (num_pages, h, page, d)),
             "selected": _history(c, cached, rows, groups, max_pages * page, gen)}
    qkv = tuple(_normal(gen, (state["total"], h, d), s) for s in (c["scale"], c["scale"], 1.0))
    return dict(state, step=step, cache=cache, history=cache["selected"].clone(), qkv=qkv)


# ---- the plain forms ---------------------------------------------------------------------------------------------------------

def _plain_append(tables, counts, total):
    """Row r has ``lengths[r]`` tokens and gets ``counts[r]`` more.  The k-th page needed, in row order, comes off the end of the
    list of free ones.  A row that does not fit (pool, table or ``total``) is left as it is: ``cached`` -1, slots -1."""
    bt, lengths, page = tables["block_tables"], tables["lengths"], tables["page_size"]
    rows, max_pages = bt.shape
    new = counts.clamp_min(0).long()
    ends = new.cumsum(0)
    starts = ends - new
    before = lengths.long()
    fits = (ends <= total) & (before + new <= max_pages * page)
    have = (before + page - 1) // page
    need = torch.where(fits, (before + new + page - 1) // page - have, 0)
    upto = need.cumsum(0)
    free = tables["free_count"].long()
    served = fits & ((need == 0) | (upto <= free))
    block = torch.arange(max_pages, device=bt.device)
    fresh = served[:, None] & (block >= have[:, None]) & (block < (have + need)[:, None])
    k = (upto - need)[:, None] + block - have[:, None]
    taken = tables["free_pages"][(free - 1 - k).clamp(0, tables["free_pages"].numel() - 1)]
    bt.copy_(torch.where(fresh, taken, bt))
    tables["page_refs"].scatter_add_(0, torch.where(fresh, taken, 0).reshape(-1).long(), fresh.reshape(-1).to(torch.int32))
    tables["free_count"].sub_(torch.where(served, need, 0).sum().to(torch.int32))
    lengths.add_(torch.where(served, new, 0).to(torch.int32))
    token = torch.arange(total, device=bt.device)
    row = torch.searchsorted(ends, token, right=True).clamp_max(rows - 1)
    position = before[row] + token - starts[row]
    inside = served[row] & (token < ends[row])
    position = torch.where(inside, position, 0)
    slots = torch.where(inside, bt[row, position // page].long() * page + position % page, -1)
    query_start = torch.cat([starts, ends[-1:]]).clamp_max(total).to(torch.int32)
    return {"query_start": query_start, "cached": torch.where(served, before, -1).to(torch.int32), "slots": slots}


def _plain_attend(cache, tables, step, q, k, v, exempt, most, longest):
    """Every row padded to ``most`` queries and ``longest`` keys."""
    page, lengths, cached = tables["page_size"], tables["lengths"], step["cached"]
    n_tok, h, d = q.shape
    slots = step["slots"]
    cache["k"][slots // page, :, slots % page] = k
    cache["v"][slots // page, :, slots % page] = v
    pages = tables["block_tables"][:, : -(-longest // page)].clamp_min(0).long()
    rows = pages.shape[0]
    j = torch.arange(pages.shape[1] * page, device=q.device)
    there = (j < lengths[:, None])[:, None, :, None]

    def gathered(pool):
        x = pool[pages].permute(0, 2, 1, 3, 4).reshape(rows, h, -1, d)
        return torch.where(there, x.float(), 0.0)

    i = torch.arange(most, device=q.device)
    start = step["query_start"][:-1].long()
    token = (start[:, None] + i).clamp_max(n_tok - 1)
    real = i < (step["query_start"][1:].long() - start)[:, None]
    logits = torch.matmul(q[token].permute(0, 2, 1, 3).float(), gathered(cache["k"]).transpose(-1, -2)) * (1.0 / math.sqrt(d))
    position = cached[:, None] + i
    can = ((j >= exempt) & (j < position[..., None]) & real[..., None])[:, None]
    groups = cache["selected"].shape[1]
    chosen = torch.relu(logits[:, :: h // groups]) * can
    old = torch.where(j < cached[:, None, None], cache["selected"][:, :, : j.numel()], 0.0)
    before = chosen.cumsum(2) - chosen + old[:, :, None]
    logits = torch.where((j <= position[..., None])[:, None], logits - before, -math.inf)
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    y = torch.matmul(e, gathered(cache["v"])) / e.sum(-1, keepdim=True)
    after = old + chosen.sum(2, dtype=torch.float64).float()
    held = cache["selected"][:, :, : j.numel()]
    held.copy_(torch.where((j < lengths[:, None])[:, None], after, held))
    row = torch.searchsorted(step["query_start"][1:].long(), torch.arange(n_tok, device=q.device), right=True)
    return y.permute(0, 2, 1, 3)[row, torch.arange(n_tok, device=q.device) - start[row]].to(q.dtype)


def _plain_select(logits, scores, width):
    """In 64 bits: two beams' candidates can be as near to one another as the rounding of a sum over the vocabulary."""
    b, k, v = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    total = scores.double()[..., None] + x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    best, at = torch.sort(total.reshape(b, k * v), dim=-1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    return best.float(), (at // v + torch.arange(b, device=at.device)[:, None] * k).to(torch.int32), at % v


def _plain_reorder(tables, cache, parents):
    bt, lengths, refs, page = tables["block_tables"], tables["lengths"], tables["page_refs"], tables["page_size"]
    rows, max_pages = bt.shape
    device = bt.device
    free_pages, count = tables["free_pages"], tables["free_count"]
    row, block = torch.arange(rows, device=device), torch.arange(max_pages, device=device)
    p = parents.long()
    old, old_len = bt.clone(), lengths.clone()
    held = -(-old_len // page)
    full, part = (old_len // page)[p], (old_len % page)[p]
    first = torch.full((rows,), rows, device=device).scatter_reduce(0, p, row, "amin")
    fresh = (part > 0) & (first[p] != row)
    new = torch.where(block < (full + (part > 0))[:, None], old[p], -1)
    stays = new >= 0
    stays[row, full.clamp_max(max_pages - 1)] &= ~fresh
    had = block < held[:, None]
    held_before = refs > 0
    refs.scatter_add_(0, old.clamp_min(0).reshape(-1).long(), -had.reshape(-1).to(torch.int32))
    refs.scatter_add_(0, new.clamp_min(0).reshape(-1).long(), stays.reshape(-1).to(torch.int32))
    # pages that no row has any more go to the end of the free list, lowest first
    gone = (refs == 0) & held_before
    rank = (~gone).to(torch.uint8).argsort(stable=True)
    n_gone = gone.sum()
    at = torch.arange(rank.numel(), device=device)
    target = torch.where(at < n_gone, count.long() + at, free_pages.numel())
    padded = torch.cat([free_pages, free_pages.new_zeros(1)]).scatter_(0, target.clamp_max(free_pages.numel()), rank.to(torch.int32))
    free_pages.copy_(padded[:-1])
    count.add_(n_gone.to(torch.int32))
    nth = fresh.long().cumsum(0) - 1
    page_of = free_pages[(count.long() - 1 - nth).clamp_min(0)]
    source = old[p, full.clamp_max(max_pages - 1)]
    new[row, full.clamp_max(max_pages - 1)] = torch.where(fresh, page_of, new[row, full.clamp_max(max_pages - 1)])
    refs.scatter_add_(0, torch.where(fresh, page_of, 0).long(), fresh.to(torch.int32))
    count.sub_(fresh.sum().to(torch.int32))
    bt.copy_(new)
    lengths.copy_(old_len[p])
    src, dst = torch.where(fresh, source, -1), torch.where(fresh, page_of, -1)
    # the tokens of the page that is being filled, and the history
    t = torch.arange(page, device=device)
    moved = (fresh[:, None] & (t < part[:, None]))[:, None, :, None]
    s, to = src.clamp_min(0).long(), torch.where(fresh, dst, new[:, 0]).long()      # without a copy: a row's first page, as it is
    for pool in (cache["k"], cache["v"]):
        pool[to] = torch.where(moved, pool[s], pool[to])
    sel = cache["selected"]
    mine = (torch.arange(sel.shape[2], device=device) < lengths[:, None])[:, None]
    sel.copy_(torch.where(mine, sel[p], sel))
    return {"copies": torch.stack([src, dst], 1)}


# ---- one pass ----------------------------------------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    with torch.no_grad():
        if c["kind"] == "select":
            if own:
                return list(_framework()[1].beam_select(state["logits"], state["scores"], c["width"]))
            return list(_plain_select(state["logits"], state["scores"], c["width"]))
        tables = state["tables"]
        if c["kind"] == "tables":                              # one more step from the same state: it goes back, then on
            state["storage"].copy_(state["saved"])
            if own:
                step = _framework()[0].append_tokens(tables, state["counts"], state["total"], max_length=state["longest"],
                                                max_count=state["most"])
            else:
                step = _plain_append(tables, state["counts"], state["total"])
            return [step["query_start"], step["cached"], step["slots"], state["storage"]]
        cache = state["cache"]
        cache["selected"].copy_(state["history"])
        if c["kind"] == "attend":                              # a layer of the step; its history goes back, then on
            if own:
                y = _framework()[0].paged_attention(cache, tables, state["step"], *state["qkv"], exempt=c["exempt"])
            else:
                y = _plain_attend(cache, tables, state["step"], *state["qkv"], c["exempt"], state["most"], state["longest"])
            return [y, cache["k"], cache["v"], cache["selected"]]
        state["storage"].copy_(state["saved"])
        if own:
            paged = _framework()[0]
            moves = paged.reorder_rows(tables, state["parents"])
            paged.move_rows(cache, moves)
        else:
            moves = _plain_reorder(tables, cache, state["parents"])
        return [moves["copies"], state["storage"], cache["k"], cache["v"], cache["selected"]]


def work(case):
    c = case
    if c["kind"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "fp32" else 2) + 16 * c["groups"] * c["width"], "flops": 3 * n}
    if c["kind"] == "reorder":
        rng = random.Random(c["ragged"])
        tokens = [c["tokens"] if c["groups"] == 1 else rng.randint(1, 2 * c["tokens"]) for _ in range(c["groups"])]
        g = c["heads"] if c["per_head"] else 1
        rows, pages = sum(tokens) * c["beams"], sum(-(-n // c["page"]) for n in tokens) * c["beams"]
        partial = sum(n % c["page"] for n in tokens) * c["beams"]
        # of uniform parents two thirds are new to their row, and about half of the rows get a page of their own
        move = 2 / 3 * (2 * 4 * g * rows + 8 * pages) + 0.5 * partial * 2 * 2 * 2 * c["heads"] * c["dim"]
        return {"bytes": move + 12 * c["groups"] * c["beams"], "flops": 0}
    cached, counts = _lengths(c)
    if c["kind"] == "tables":
        pages = sum(-(-(a + b) // c["page"]) - -(-a // c["page"]) for a, b in zip(cached, counts))
        return {"bytes": 8 * sum(counts) + 16 * pages + 20 * len(counts), "flops": 0}
    h, d, g = c["heads"], c["dim"], c["heads"] if c["per_head"] else 1
    pairs = sum(n * a + n * (n + 1) / 2 for a, n in zip(cached, counts))
    keys, new = sum(cached), sum(counts)
    selection = 0 if c["per_head"] else 2 * pairs * d          # a head that selects for itself has its logits already
    return {"bytes": 2 * keys * h * d * 2 + 6 * new * h * d * 2 + 8 * g * keys, "flops": 4 * pairs * h * d + selection}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    """From the definition, row by row and head by head, on numbers of 64 bits."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "tables":
        return None
    if c["kind"] == "select":
        total = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
        return [total.flatten(1).topk(c["width"], dim=1).values, None, None]
    if c["kind"] == "reorder":
        sel, want = s["history"].double(), s["history"].double()
        lengths, page = s["tables"]["lengths"].tolist(), c["page"]
        for r, p in enumerate(s["parents"].tolist()):
            want[r, :, : lengths[p]] = sel[p, :, : lengths[p]]
        return [None, None, None, None, want]
    cached, counts = _lengths(c)
    h, d, exempt, page = c["heads"], c["dim"], c["exempt"], c["page"]
    q, k, v = s["qkv"]
    selected = s["history"].double()
    groups = selected.shape[1]
    y = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (a, n) in enumerate(zip(cached, counts)):
        ids = s["tables"]["block_tables"][r, : -(-(a + n) // page)].long()
        i = torch.arange(a, a + n, device="cuda")[:, None]
        j = torch.arange(a + n, device="cuda")[None]
        start = torch.cat([selected[r, :, :a], torch.zeros(groups, n, dtype=torch.float64, device="cuda")], 1)
        history = None
        for x in range(h):
            keys, values = (torch.cat([pool[ids, x].reshape(-1, d)[:a], fresh[at:at + n, x]]).double()
                            for pool, fresh in ((s["cache"]["k"], k), (s["cache"]["v"], v)))
            z = q[at:at + n, x].double() @ keys.T / math.sqrt(d)
            if x % (h // groups) == 0:
                took = z.clamp_min(0).masked_fill((j >= i) | (j < exempt), 0.0)
                g = x // (h // groups)
                history = start[g] + took.cumsum(0) - took
                selected[r, g, : a + n] = start[g] + took.sum(0)
                del took
            z = z.sub_(history).masked_fill_(j > i, -math.inf)
            y[at:at + n, x] = torch.softmax(z, -1) @ values
            del z
        at += n
    return [y, None, None, selected]
