"""CPU restatement of the paged cache, its attention and beam selection: tables row by row in Python, attention from the
definition in 64 bits.  Test infrastructure, like ``selective_oracle``."""

import math

import torch


class Tables:
    """Block tables as lists: what ``paged.append_tokens`` and ``paged.reorder_rows`` do, one page at a time."""

    def __init__(self, rows, num_pages, page, max_pages):
        self.page, self.max_pages = page, max_pages
        self.blocks = [[] for _ in range(rows)]
        self.lengths = [0] * rows
        self.free = list(range(num_pages - 1, -1, -1))
        self.refs = [0] * num_pages

    def append(self, counts, total, max_length=None, max_count=None):
        capacity = self.max_pages * self.page
        limit = min(capacity, max_length or capacity)
        at, slots, starts, cached = 0, [-1] * total, [], []
        full = False
        free, taken = list(self.free), 0
        for r, count in enumerate(counts):
            count = max(count, 0)
            starts.append(min(at, total))
            before, at = self.lengths[r], at + count
            fits = at <= total and before + count <= limit and count <= (max_count or capacity)
            need = -(-(before + count) // self.page) - -(-before // self.page) if fits else 0
            if need and (full or taken + need > len(free)):
                full, fits = True, False
            if not fits:
                cached.append(-1)
                continue
            for _ in range(need):
                page = free[len(free) - 1 - taken]
                taken += 1
                self.refs[page] += 1
                self.blocks[r].append(page)
            cached.append(before)
            self.lengths[r] = before + count
            for i in range(count):
                p = before + i
                slots[starts[r] + i] = self.blocks[r][p // self.page] * self.page + p % self.page
        self.free = free[:len(free) - taken]
        return starts + [min(at, total)], cached, slots

    def reorder(self, parents):
        rows = len(parents)
        old, old_lengths = [list(b) for b in self.blocks], list(self.lengths)
        for blocks in old:
            for page in blocks:
                self.refs[page] -= 1
        wants, keeps = [], {}
        for r, p in enumerate(parents):
            self.blocks[r], self.lengths[r] = [], 0
            if not 0 <= p < rows:
                continue
            full, part = divmod(old_lengths[p], self.page)
            self.blocks[r], self.lengths[r] = old[p][:full], old_lengths[p]
            for page in self.blocks[r]:
                self.refs[page] += 1
            if part and p not in keeps:
                keeps[p] = r
                self.blocks[r].append(old[p][full])
                self.refs[old[p][full]] += 1
            elif part:
                wants.append((r, old[p][full]))
        held = {page for blocks in old for page in blocks}
        self.free += sorted(page for page in held if self.refs[page] == 0)
        copies = [(-1, -1)] * rows
        for r, source in wants:
            if self.free:
                page = self.free.pop()
                copies[r] = (source, page)
                self.blocks[r].append(page)
                self.refs[page] += 1
            else:
                for page in self.blocks[r]:
                    self.refs[page] -= 1
                self.blocks[r], self.lengths[r] = [], 0
        return copies


def attend(q, k, v, history, cached, exempt, per_head):
    """New queries of one row, (n, H, D), over all of its keys and values (cached + n, H, D); ``history`` (G, cached).  Everything in
    64 bits.  Returns y (n, H, D), the history after (G, cached + n), and bounds on what bf16 operands of the products may be off:
    one for y with the probabilities and the selection inside a 128-query tile rounded to bf16, one for the history."""
    n, h, d = q.shape
    t = cached + n
    q, k, v = q.double(), k.double(), v.double()
    i, j = torch.arange(cached, t)[:, None], torch.arange(t)[None]
    can = (j < i) & (j >= exempt)
    logits = torch.einsum("nhd,thd->hnt", q, k) / math.sqrt(d)
    sizes = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()) / math.sqrt(d)
    heads = range(h) if per_head else [0]
    start = torch.cat([history.double(), torch.zeros(history.shape[0], n, dtype=torch.float64)], 1)
    y, y_off = torch.empty(n, h, d, dtype=torch.float64), torch.empty(n, h, d, dtype=torch.float64)
    after, after_off = start.clone(), torch.empty_like(start)
    took, before, inside = {}, {}, {}
    for g, x in enumerate(heads):
        took[x] = logits[x].clamp_min(0) * can
        run = took[x].cumsum(0) - took[x]
        before[x] = start[g] + run
        # what the queries of the same tile before it have selected: rounded to bf16 (half a step, 2^-8 of it)
        first = (i[:, 0] // 128 * 128 - cached).clamp_min(0)
        inside[x] = run - run[first]
        after[g] = start[g] + took[x].sum(0)
        # 32-bit sums: of D products a logit (the tensor cores may cut where the CPU rounds: a whole step), then of n logits
        after_off[g] = 2.0 ** -23 * ((d + n + 2) * (sizes[x] * can).sum(0) + after[g]) + 1e-30
    for x in range(h):
        s = x if per_head else 0
        z = (logits[x] - before[s]).masked_fill(j > i, -math.inf)
        p = torch.softmax(z, -1)
        y[:, x] = p @ v[:, x]
        # relative error of a probability: the logit's own (32-bit sums of D products and of the history), its rounding, and the
        # selection's; y = sum p v / sum p has it once above and once below the line
        small = 2.0 ** -23 * ((d + 4) * sizes[x] + 4 * before[s]) + 2.0 ** -20
        rel = torch.expm1(2.0 ** -8 * inside[s] + small).masked_fill((j > i) | torch.isinf(before[s]), 0.0)      # (no weight at all)
        y_off[:, x] = (p * (rel + 2.0 ** -8 * (1 + rel))) @ v[:, x].abs() + (p * rel).sum(-1, keepdim=True) * y[:, x].abs()
    y_off = 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * y_off + 1e-30             # the output's own rounding
    return y, after, y_off, after_off


def select(logits, scores, width):
    """(groups, beams, vocab) in 64 bits; a score that is not finite counts as -inf."""
    groups, beams, vocab = logits.shape
    lse = torch.logsumexp(logits.double(), -1, keepdim=True)
    base = scores.double()[..., None] - lse
    total = torch.where(torch.isfinite(base), base + logits.double(), -math.inf)
    total = torch.where(torch.isnan(total), -math.inf, total).reshape(groups, beams * vocab)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    return best, at // vocab + torch.arange(groups)[:, None] * beams, at % vocab
