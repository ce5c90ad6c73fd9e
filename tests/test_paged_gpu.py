"""The paged cache against its oracle: tables page by page, attention row by row in 64 bits with derived bounds, rows that become
copies, and a run of them together."""

import random

import pytest
import torch

import paged_oracle
from selective_attention_b200 import _lib, kernels, mixers, paged

pytestmark = pytest.mark.gpu


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _same_tables(t, want):
    blocks = t["block_tables"].cpu().tolist()
    assert t["lengths"].tolist() == want.lengths
    for r, held in enumerate(want.blocks):
        assert blocks[r][:len(held)] == held, r
    n = int(t["free_count"])
    assert t["free_pages"].tolist()[:n] == want.free and t["page_refs"].tolist() == want.refs


def _both(rows, num_pages, page, max_pages, heads=2):
    return paged.begin_tables(rows, num_pages, page, max_pages, heads), paged_oracle.Tables(rows, num_pages, page, max_pages)


def _append(t, want, counts, total, **bounds):
    step = paged.append_tokens(t, _ints(counts), total, **bounds)
    starts, cached, slots = want.append(counts, total, **bounds)
    assert step["query_start"].tolist() == starts and step["cached"].tolist() == cached and step["slots"].tolist() == slots
    _same_tables(t, want)
    return step


# ---- tables ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,page,most", [(1, 16, 300), (3, 256, 500), (64, 16, 3), (200, 64, 70), (300, 16, 40), (1025, 32, 20), (4096, 16, 5)])
def test_steps_equal_the_oracle(rows, page, most):
    rng = random.Random(rows)
    max_pages = -(-6 * most // page)
    t, want = _both(rows, rows * max_pages, page, max_pages)
    for _ in range(4):
        counts = [rng.choice([0, 1, 1, rng.randint(-2, most)]) for _ in range(rows)]
        total = sum(max(c, 0) for c in counts)
        _append(t, want, counts, total)
    counts = [1] * rows
    _append(t, want, counts, rows, max_count=1)


def test_a_long_step_writes_its_slots_from_many_blocks():
    t, want = _both(5, 9000, 16, 2000)
    _append(t, want, [3, 9000, 0, 12345, 17], 21400)              # 35 tokens behind the last row
    _append(t, want, [1, 1, 1, 1, 1], 5)


def test_rows_that_do_not_fit_are_left_as_they_were():
    t, want = _both(6, 10, 16, 4)
    _append(t, want, [40, 0, 65, 16, 1, 20], 142)                  # row 2: its table
    _append(t, want, [1, 33, 1, 48, 15, 1], 99)                    # the pool gives out in row 3: nothing for rows that need a page
    _append(t, want, [1, 1, 1, 1, 1, 1], 4)                        # total
    _append(t, want, [9, 1, 1, 1, 1, 2], 15, max_length=40)        # rows 0 and 1
    _append(t, want, [1, 2, 1, 1, 1, 3], 9, max_count=1)           # rows 1 and 5
    _append(t, want, [2 ** 30] * 6, 50)
    _append(t, want, [0] * 6, 0)
    _append(t, want, [-5] * 6, 3)


@pytest.mark.parametrize("rows,page,num_pages", [(4, 16, 64), (33, 32, 200), (700, 16, 9000), (1500, 16, 9000)])
def test_rows_become_copies_as_in_the_oracle(rows, page, num_pages):
    rng = random.Random(rows + page)
    t, want = _both(rows, num_pages, page, 8)
    for trial in range(5):
        counts = [rng.choice([0, 1, page, rng.randint(0, page)]) for _ in range(rows)]
        _append(t, want, counts, sum(counts))
        near = trial % 2 == 0                                     # beams of one request, or any row
        parents = [max(-1, r // 4 * 4 + rng.randint(0, 3) if near else rng.randint(-2, rows)) for r in range(rows)]
        parents = [p if p < rows or not near else rows - 1 for p in parents]
        moves = paged.reorder_rows(t, _ints(parents))
        assert [tuple(x) for x in moves["copies"].tolist()] == want.reorder(parents)
        _same_tables(t, want)
        assert all((row[len(held):] == [-1] * (8 - len(held))) for row, held in zip(t["block_tables"].tolist(), want.blocks))


@pytest.mark.parametrize("rows,max_pages", [(1, 33), (3, 64), (5, 1000), (100, 70), (129, 65)])
def test_copies_of_rows_of_many_pages(rows, max_pages):
    rng = random.Random(rows)
    t, want = _both(rows, rows * max_pages, 16, max_pages)
    counts = [rng.randint(1, 16 * max_pages) for _ in range(rows - 1)] + [16 * max_pages - 1]
    _append(t, want, counts, sum(counts))
    for _ in range(3):
        parents = [rng.randint(-1, rows - 1) for _ in range(rows - 1)] + [rows - 1]
        moves = paged.reorder_rows(t, _ints(parents))
        assert [tuple(x) for x in moves["copies"].tolist()] == want.reorder(parents)
        _same_tables(t, want)


def test_copies_in_a_full_pool():
    t, want = _both(6, 8, 16, 4)
    _append(t, want, [20, 20, 40, 0, 0, 0], 80)                    # 7 of 8 pages
    for parents in ([0, 0, 2, 0, 2, 2], [0, 1, 2, 3, 4, 5], [1, 1, 1, 1, 1, 1], [5, 4, -1, 2, 1, 0]):
        moves = paged.reorder_rows(t, _ints(parents))
        assert [tuple(x) for x in moves["copies"].tolist()] == want.reorder(parents)
        _same_tables(t, want)
    want.reorder([-1] * 6)
    paged.reorder_rows(t, _ints([-1] * 6))
    _same_tables(t, want)
    assert int(t["free_count"]) == 8


@pytest.mark.parametrize("rows,free", [(6, 0), (6, 2), (40, 7), (1500, 700), (300, 299), (300, 300)])
def test_rows_that_are_lost_are_counted(rows, free):
    """Copies of one row that need a page each, in a pool that has `free` of them; then with nothing to copy."""
    t, want = _both(rows, 2 + free, 16, 2)
    _append(t, want, [21] + [0] * (rows - 1), 21)
    moves = paged.reorder_rows(t, _ints([0] * rows))
    assert [tuple(x) for x in moves["copies"].tolist()] == want.reorder([0] * rows)
    _same_tables(t, want)
    assert moves["lost"].dtype == torch.int32 and moves["lost"].tolist() == [max(rows - 1 - free, 0)]
    assert int((t["lengths"] == 0).sum()) == max(rows - 1 - free, 0)
    moves = paged.reorder_rows(t, _ints(list(range(rows))))
    assert moves["lost"].tolist() == [0] and (moves["copies"] == -1).all()
    moves = paged.reorder_rows(t, _ints([-1] * rows))             # given back, not lost
    assert moves["lost"].tolist() == [0] and int(t["free_count"]) == 2 + free


# ---- attention ---------------------------------------------------------------------------------------------------------------

class Served:
    """A paged layer beside what the oracle knows of it: every row's keys, values and history."""

    def __init__(self, rows, heads, dim, page, max_pages, num_pages, per_head=False, exempt=1, scale=1.0, seed=0):
        self.gen = torch.Generator().manual_seed(seed)
        self.t, self.want = _both(rows, num_pages, page, max_pages, heads)
        self.slot = mixers.SelectiveAttentionSlot(heads, max_pages * page, exempt=exempt, per_head=per_head)
        self.cache = self.slot.begin_pages(self.t, dim)
        for x in self.cache.values():                             # what stands in pages and histories that nobody owns
            x.fill_(float("nan"))
        self.heads, self.dim, self.exempt, self.per_head, self.scale = heads, dim, exempt, per_head, scale
        empty = (torch.zeros(0, heads, dim), torch.zeros(0, heads, dim), torch.zeros(heads if per_head else 1, 0, dtype=torch.float64))
        self.rows = [empty] * rows

    def tokens(self, n):
        q, k = (torch.randn(n, self.heads, self.dim, generator=self.gen) * self.scale for _ in range(2))
        return tuple(x.bfloat16() for x in (q, k, torch.randn(n, self.heads, self.dim, generator=self.gen)))

    def expect(self, counts, starts, cached, q, k, v, y):
        worst = 0.0
        for r, n in enumerate(counts):
            if cached[r] < 0 or n < 1:
                continue
            a = starts[r]
            keys, values, history = self.rows[r]
            assert keys.shape[0] == cached[r]
            keys, values = (torch.cat([old, new[a:a + n].float()]) for old, new in ((keys, k), (values, v)))
            want, history, off, _ = paged_oracle.attend(q[a:a + n].float(), keys, values, history, cached[r], self.exempt, self.per_head)
            miss = ((y[a:a + n].double().cpu() - want).abs() / off).max().item()
            assert miss <= 1.0, (r, n, cached[r], miss)
            worst = max(worst, miss)
            self.rows[r] = (keys, values, history)
        return worst

    def histories(self):
        got = self.cache["selected"].cpu()
        for r, (keys, _, history) in enumerate(self.rows):
            n = keys.shape[0]
            if n:
                # every step adds its own rounding: the oracle's bound is of the last one, so the whole is held relatively
                err = (got[r, :, :n].double() - history).abs() / (history + self.scale ** 2)
                assert err.max().item() <= 2.0 ** -23 * (self.dim + 2 * n + 64), r
            assert torch.isnan(got[r, :, n:]).all(), r             # behind the last token nothing is written

    def pools(self):
        """The pages hold the rows' keys and values, everything else is as it was."""
        for name, i in (("k", 0), ("v", 1)):
            got = self.cache[name].cpu()
            seen = torch.isnan(got)
            for r, row in enumerate(self.rows):
                for p in range(row[0].shape[0]):
                    page, at = self.want.blocks[r][p // self.t["page_size"]], p % self.t["page_size"]
                    assert torch.equal(got[page, :, at].float(), row[i][p]), (name, r, p)
                    seen[page, :, at] = True
            assert seen.all()

    def step(self, counts, total=None, fused=False, **bounds):
        n = sum(max(c, 0) for c in counts) if total is None else total
        step = _append(self.t, self.want, counts, n, **bounds)
        q, k, v = self.tokens(n)
        if fused:                                                  # slots of a projection's output, and a head order of its own
            qkv = torch.stack([q, k, v], 1).cuda()
            args = [qkv[:, i] for i in range(3)]
            args[0] = args[0].transpose(0, 1).contiguous().transpose(0, 1)
        else:
            args = [x.cuda() for x in (q, k, v)]
        y = self.slot.attend_pages(*args, self.cache, self.t, step)
        assert y.shape == (n, self.heads, self.dim) and y.dtype == torch.bfloat16
        unserved = step["slots"].cpu() < 0
        assert (y.cpu()[unserved] == 0).all()
        worst = self.expect(counts, step["query_start"].tolist(), step["cached"].tolist(), q, k, v, y)
        self.histories()
        assert _lib.device_status() == 0
        return worst


SHAPES = [(2, 64, 16, False), (3, 64, 32, True), (4, 128, 64, False), (2, 128, 128, True), (1, 64, 256, False), (5, 128, 16, False)]


@pytest.mark.parametrize("heads,dim,page,per_head", SHAPES)
def test_single_tokens_of_ragged_rows(heads, dim, page, per_head, achieved):
    rows, worst = 7, 0.0
    s = Served(rows, heads, dim, page, -(-700 // page), rows * (-(-700 // page)), per_head, exempt=2)
    s.step([1, 0, 600, 127, 128, 129, 16])                         # prompts (row 0: a single token from the start)
    for counts in ([1] * rows, [1, 1, 0, 1, 1, 0, 1], [1] * rows):
        worst = max(worst, s.step(counts, max_count=1, fused=True))
    s.pools()
    achieved(f"paged single tokens H={heads} D={dim} page={page}", share_of_bound=worst)


@pytest.mark.parametrize("heads,dim,page,per_head", SHAPES)
def test_chunks_of_ragged_rows(heads, dim, page, per_head, achieved):
    rows, worst = 6, 0.0
    s = Served(rows, heads, dim, page, -(-1100 // page), rows * (-(-1100 // page)), per_head, exempt=1, scale=0.5, seed=1)
    for counts in ([300, 1, 128, 0, 257, 2], [5, 1, 1, 129, 130, 126], [400, 127, 0, 1, 300, 2]):
        worst = max(worst, s.step(counts, fused=True))
    s.pools()
    achieved(f"paged chunks H={heads} D={dim} page={page}", share_of_bound=worst)


@pytest.mark.parametrize("heads,dim,page,per_head", SHAPES)
def test_rows_of_few_tokens(heads, dim, page, per_head, achieved):
    """Two to eight tokens of a row: across pages and key tiles, alone and beside rows of more."""
    rows = 7
    s = Served(rows, heads, dim, page, -(-800 // page), rows * (-(-800 // page)), per_head, exempt=2, seed=5)
    s.step([60, 0, 600, 126, 127, 121, 16])
    worst = max(s.step(counts, max_count=8, fused=True) for counts in ([2, 3, 8, 4, 1, 7, 0], [5] * rows, [8, 1, 2, 3, 0, 5, 6]))
    worst = max(worst, s.step([1, 9, 2, 8, 3, 30, 7], fused=True), s.step([2, 1, 0, 0, 0, 0, 3], total=8), s.step([1] * rows, max_count=1))
    s.pools()
    achieved(f"paged few tokens H={heads} D={dim} page={page}", share_of_bound=worst)


@pytest.mark.parametrize("heads,dim,per_head,rows", [(4, 64, False, 1), (2, 64, True, 2), (3, 128, False, 2), (1, 128, True, 1)])
def test_few_tokens_after_many(heads, dim, per_head, rows, achieved):
    """Rows whose keys are cut into pieces, with new tokens on both sides of a cut."""
    s = Served(rows, heads, dim, 32, 70, 70 * rows, per_head, exempt=16, scale=0.4, seed=6)
    worst = s.step([2045 - 256 * r for r in range(rows)])         # the first 8 lie on both sides of a multiple of 128
    for n in (8, 5, 1, 8, 7, 2):
        worst = max(worst, s.step([n] * rows, max_count=8))
    s.pools()
    achieved(f"paged few tokens after 2,000 H={heads} D={dim}", share_of_bound=worst)


@pytest.mark.parametrize("heads,dim,per_head,first,chunk", [
    (2, 64, False, 5000, 40),                                     # few tiles after many keys: pieces of a walk
    (16, 64, False, 300, 1500), (32, 64, False, 100, 1450), (32, 64, True, 100, 1300),      # many tiles: one head a CTA, and two
    (16, 64, False, 2000, 500), (16, 64, True, 2300, 500),        # walks in pieces of which there are two waves
    (12, 64, False, 1, 1700), (5, 64, False, 777, 1601), (8, 128, False, 500, 1300), (16, 64, True, 129, 1200), (3, 128, True, 3000, 129)])
def test_one_row_prompt_and_chunk(heads, dim, per_head, first, chunk, achieved):
    s = Served(1, heads, dim, 64, -(-(first + chunk + 3) // 64), 120, per_head, exempt=16, scale=0.3, seed=2)
    worst = max(s.step([first]), s.step([chunk]), s.step([1], total=3), s.step([1]))
    s.pools()
    achieved(f"paged prompt and chunk H={heads} D={dim} {first}+{chunk}", share_of_bound=worst)


@pytest.mark.parametrize("per_head", [False, True])
def test_chunks_of_many_tiles(per_head, achieved):
    """Several rows whose tiles are more than the SMs: two heads a CTA."""
    s = Served(3, 16, 64, 32, 60, 150, per_head, exempt=3, scale=0.4, seed=8)
    worst = max(s.step([900, 33, 700]), s.step([700, 1, 810]), s.step([640, 500, 200]))
    s.pools()
    achieved(f"paged chunks of many tiles per_head={per_head}", share_of_bound=worst)


@pytest.mark.parametrize("heads,dim,per_head", [(16, 64, False), (32, 64, False), (16, 64, True), (16, 128, False), (8, 128, True)])
def test_a_step_with_room_for_more_tokens(heads, dim, per_head):
    """The kernels are chosen for `total` tokens, the plan is made for those that there are."""
    s = Served(2, heads, dim, 64, 45, 70, per_head, exempt=2, scale=0.4, seed=10)
    s.step([1200, 30])
    s.step([150, 0], total=2600)
    s.step([0, 40], total=2000, max_count=1300)
    s.step([5, 9], total=1900)
    s.pools()
    s = Served(1, heads, dim, 64, 45, 45, per_head, exempt=2, scale=0.4, seed=11)
    s.step([1200])
    s.step([150], total=1650)
    s.step([3], total=1400)
    s.pools()


def test_rows_that_are_not_served():
    s = Served(5, 4, 64, 16, 12, 16, scale=0.5)
    s.step([100, 20, 0, 5, 1])
    s.step([1, 80, 1, 1, 1])                                      # row 1 exhausts the pool: rows 2 and on where they need a page
    s.step([1, 1, 1, 1, 1], total=3, max_count=1)                 # rows 3 and 4 are outside the step
    s.step([1, 2, 1, 1, 1], total=9, max_count=1)                 # row 1 gets more than the bound; three tokens behind the last row
    s.step([150, 1, 3, 1, 1])                                     # row 0: its table
    s.step([0] * 5, total=4)
    s.pools()


@pytest.mark.parametrize("exempt", [2 ** 31, 2 ** 32 + 1])
def test_a_layer_in_which_nothing_is_selected(exempt):
    """More exempt positions than 32 bits count: plain causal attention, in a prompt, a chunk and single tokens, paged and dense."""
    s = Served(2, 4, 64, 16, 20, 40, exempt=exempt, scale=0.5)
    for counts in ([200, 30], [1, 1], [3, 60], [5, 1]):
        s.step(counts)
    assert (s.cache["selected"][0, :, :209] == 0).all()
    q, k, v = (x.transpose(0, 1)[None].cuda() for x in s.tokens(150))
    y = kernels.selective_attention_forward(q, k, v, exempt=exempt)[0]
    assert torch.equal(y, kernels.selective_attention_forward(q, k, v, exempt=150)[0])


def test_outputs_equal_the_dense_cache():
    """The same numbers through the dense cache: rows of one length, a prompt, a chunk and single tokens."""
    gen = torch.Generator().manual_seed(5)
    rows, h, d, lengths = 2, 4, 64, (200, 131, 1, 1)
    slot = mixers.SelectiveAttentionSlot(h, 512)
    t = paged.begin_tables(rows, 64, 32, 16, h)
    cache, dense = slot.begin_pages(t, d), None
    for n in lengths:
        q, k, v = (torch.randn(rows, h, n, d, generator=gen).bfloat16().cuda() for _ in range(3))
        step = paged.append_tokens(t, _ints([n] * rows), rows * n)
        packed = [x.transpose(1, 2).reshape(rows * n, h, d) for x in (q, k, v)]
        y = slot.attend_pages(*packed, cache, t, step).view(rows, n, h, d).transpose(1, 2)
        if dense is None:
            want, dense = slot.begin_cache(q, k, v)
        else:
            want = slot.extend_cache(q, k, v, dense) if n > 1 else slot.step_cache(q, k, v, dense)
        # two roundings of the output (2^-8 each) and the probabilities' in an order of their own
        torch.testing.assert_close(y.float(), want.float(), atol=2.0 ** -6, rtol=2.0 ** -6)
    n = sum(lengths)
    torch.testing.assert_close(cache["selected"][:, :, :n], dense["selected"][:, :, :n], atol=1e-4, rtol=1e-5)


def test_tokens_of_any_strides():
    """Broadcast heads and tokens, rows at odd addresses, other types: as their contiguous bf16 form."""
    s = _prefix(4, 64, False, [70, 300])
    caches = [{name: x.clone() for name, x in s.cache.items()} for _ in range(6)]
    step = paged.append_tokens(s.t, _ints([33, 1]), 34)
    q, k, v = (x.cuda() for x in s.tokens(34))
    k, v = k[:, :1].expand(-1, 4, -1), v[:1].expand(34, -1, -1)
    wide = torch.zeros(34, 4, 67, device="cuda", dtype=torch.bfloat16)
    wide[:, :, 3:] = q
    forms = [(q, k.contiguous(), v.contiguous()), (q, k, v), (wide[:, :, 3:], k, v), (q.float(), k.float(), v.half()),
             (q.transpose(1, 2).contiguous().transpose(1, 2), k, v), (q[:, :1].expand(-1, 4, -1), k, v)]
    ys = [paged.paged_attention(cache, s.t, step, *x) for cache, x in zip(caches, forms)]
    for y, cache in zip(ys[1:5], caches[1:5]):
        assert torch.equal(y, ys[0])
        for name in ("k", "v", "selected"):
            assert torch.equal(torch.nan_to_num(cache[name]), torch.nan_to_num(caches[0][name]))
    assert torch.isfinite(ys[5].float()).all()


@pytest.mark.parametrize("counts", [[33, 1], [1, 1], [5, 1]])
def test_tokens_of_heads_that_share_them(counts):
    """q, k, v of one head for all of them (a stride of 0 over heads), or of one token for all: as when every head has its copy."""
    s = _prefix(4, 64, False, [70, 300])
    n = sum(counts)
    step = paged.append_tokens(s.t, _ints(counts), n, max_count=max(counts))
    q, k, v = (x.cuda() for x in s.tokens(n))
    head = lambda x: x[:, :1].expand(-1, 4, -1)                    # noqa: E731
    token = lambda x: x[:1].expand(n, -1, -1)                      # noqa: E731
    both = lambda x: x[:1, :1].expand(n, 4, -1)                    # noqa: E731
    for form in ((head(q), k, v), (q, head(k), v), (q, k, head(v)), (token(q), token(k), token(v)), (both(q), both(k), both(v)),
                 (head(q).float(), head(k).half(), token(v).float())):
        shared, own = ({name: x.clone() for name, x in s.cache.items()} for _ in range(2))
        y = paged.paged_attention(shared, s.t, step, *form)
        want = paged.paged_attention(own, s.t, step, *(x.bfloat16().contiguous().clone() for x in form))
        assert torch.equal(y, want) and torch.isfinite(y.float()).all() and (y != 0).any()
        for name in ("k", "v", "selected"):
            assert torch.equal(torch.nan_to_num(shared[name]), torch.nan_to_num(own[name])), name


@pytest.mark.parametrize("heads,per_head", [(2, False), (16, False), (4, True)])
def test_keys_that_were_taken_out(heads, per_head):
    """Keys whose history their owner has made infinite have no weight: as if they were not there."""
    lengths = [500, 200, 64]
    s = _prefix(heads, 64, per_head, lengths)
    gone = slice(16, 400)                                          # whole tiles and pages of row 0, a part of the others'
    for r, n in enumerate(lengths):
        s.cache["selected"][r, :, gone.start:min(gone.stop, n)] = float("inf")
        keys, values, history = s.rows[r]
        s.rows[r] = (keys, values, torch.cat([history[:, :16], torch.full_like(history[:, gone], float("inf")), history[:, 400:]], 1))
    for counts in ([1, 1, 1], [130, 40, 500], [1, 1, 1], [3, 8, 1]):
        n = sum(counts)
        step = _append(s.t, s.want, counts, n)
        q, k, v = s.tokens(n)
        y = s.slot.attend_pages(q.cuda(), k.cuda(), v.cuda(), s.cache, s.t, step)
        s.expect(counts, step["query_start"].tolist(), step["cached"].tolist(), q, k, v, y)
        got = s.cache["selected"].cpu()
        for r, (_, _, history) in enumerate(s.rows):
            assert torch.equal(torch.isinf(got[r, :, :history.shape[1]]), torch.isinf(history))


def test_many_rows():
    """More rows than a thread has in the plan's sums, and more walks and pieces than CTAs that are resident."""
    rows, rng = 1100, random.Random(8)
    s = Served(rows, 2, 64, 16, 10, 5 * rows, scale=0.7, seed=9)
    s.step([rng.choice([0, 1, 2, 3, 40]) for _ in range(rows)])
    s.step([rng.choice([0, 1]) for _ in range(rows)], max_count=1)
    s.step([rng.choice([0, 1, 1, 5]) for _ in range(rows)])


def test_pools_beyond_32_bit_offsets():
    """Pages whose elements lie beyond 2^31: the same numbers as in a small pool."""
    h, d, page = 16, 64, 32
    outs = []
    for num_pages in (80, 70000):                                  # 70,000 pages of 32 x 1,024 elements
        t = paged.begin_tables(2, num_pages, page, 40, h)
        t["free_pages"].copy_(torch.arange(num_pages, dtype=torch.int32))          # the last pages first
        cache = paged.begin_pages(t, d)
        gen = torch.Generator().manual_seed(4)
        got = []
        for counts in ([500, 77], [1, 1], [200, 40], [1, 1]):
            step = paged.append_tokens(t, _ints(counts), sum(counts))
            x = [torch.randn(sum(counts), h, d, generator=gen).bfloat16().cuda() for _ in range(3)]
            got.append(paged.paged_attention(cache, t, step, *x))
        moves = paged.reorder_rows(t, _ints([0, 0]))
        paged.move_rows(cache, moves)
        step = paged.append_tokens(t, _ints([1, 1]), 2)
        got.append(paged.paged_attention(cache, t, step, *(torch.randn(1, h, d, generator=gen).bfloat16().cuda().repeat(2, 1, 1) for _ in range(3))))
        assert torch.equal(got[-1][0], got[-1][1]) and (num_pages == 80 or int(t["block_tables"].max()) == num_pages - 1)
        outs.append(got + [cache["selected"]])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_pages_outside_the_pool_read_as_zeros():
    """A table that its owner has damaged: nothing outside the pools is read or written."""
    h, d = 2, 64
    for n, most in ((1, 1), (40, 40), (6, 6)):
        t = paged.begin_tables(2, 16, 16, 8, h)
        cache = paged.begin_pages(t, d)
        first = paged.append_tokens(t, _ints([64, 64]), 128)
        x = [torch.randn(128, h, d).bfloat16().cuda() for _ in range(3)]
        paged.paged_attention(cache, t, first, *x)
        step = paged.append_tokens(t, _ints([n, n]), 2 * n, max_count=most)
        t["block_tables"][1, 1] = 10 ** 6
        t["block_tables"][1, 2] = -7
        step["slots"][-1] = 10 ** 9
        y = paged.paged_attention(cache, t, step, *(z[:2 * n].contiguous() for z in x))
        torch.cuda.synchronize()
        assert torch.isfinite(y.float()).all() and _lib.device_status() == 0


def test_arguments_that_are_refused():
    t = paged.begin_tables(2, 16, 16, 8, 2)
    cache = paged.begin_pages(t, 64)
    step = paged.append_tokens(t, _ints([3, 4]), 7)
    x = torch.zeros(7, 2, 64, device="cuda", dtype=torch.bfloat16)
    for bad, match in (((x[:6], x, x), "the step's tokens"), ((x, x[:, :1], x), "the step's tokens"), ((x, x, x.cpu()), "CUDA"),
                       ((x.long(), x, x), "float16")):
        with pytest.raises(ValueError, match=match):
            paged.paged_attention(cache, t, step, *bad)
    with pytest.raises(ValueError, match="num_pages"):
        paged.paged_attention(dict(cache, k=cache["k"][:8]), t, step, x, x, x)
    with pytest.raises(ValueError, match="selected"):
        paged.paged_attention(dict(cache, selected=cache["selected"][:, :, :64]), t, step, x, x, x)
    with pytest.raises(ValueError, match="bf16"):
        paged.paged_attention(dict(cache, k=cache["k"].half()), t, step, x, x, x)
    other = paged.begin_tables(2, 16, 16, 9, 2)
    with pytest.raises(ValueError, match="other tables"):
        paged.paged_attention(paged.begin_pages(other, 64), other, step, x, x, x)
    with pytest.raises(ValueError, match="counts"):
        paged.append_tokens(t, _ints([3, 4]).long(), 7)
    with pytest.raises(ValueError, match="counts"):
        paged.append_tokens(t, _ints([3, 4, 5]), 12)
    with pytest.raises(ValueError, match="parents"):
        paged.reorder_rows(t, _ints([0]))
    with pytest.raises(ValueError, match="int32"):
        paged.append_tokens(dict(t, lengths=t["lengths"].long()), _ints([3, 4]), 7)


# ---- streams and graphs ------------------------------------------------------------------------------------------------------

def _prefix(heads, dim, per_head, lengths, page=16, seed=7):
    s = Served(len(lengths), heads, dim, page, 40, 40 * len(lengths), per_head, scale=0.4, seed=seed)
    s.step(lengths)
    return s


@pytest.mark.parametrize("counts,most", [([1, 1, 1], 1), ([1, 40, 130], 130), ([2, 8, 5], 8), ([1, 7, 130], 130)])
def test_a_captured_step_is_replayed(counts, most):
    s = _prefix(4, 64, False, [100, 300, 20])
    n = sum(counts)
    q, k, v = (torch.zeros(n, 4, 64, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    device_counts = _ints([0, 0, 0])
    saved = {name: x.clone() for name, x in s.t.items() if torch.is_tensor(x)}
    history = s.cache["selected"].clone()

    def run():
        step = paged.append_tokens(s.t, device_counts, n, max_count=most)
        return step, s.slot.attend_pages(q, k, v, s.cache, s.t, step)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()                                                      # nothing is appended: all counts are zero
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, y = run()
    for name, x in saved.items():
        assert torch.equal(s.t[name], x), name
    assert torch.equal(torch.nan_to_num(s.cache["selected"]), torch.nan_to_num(history))
    for turn in ([counts, [0, 0, 0], counts[::-1], counts]):
        tokens = s.tokens(n)
        for to, x in zip((q, k, v), tokens):
            to.copy_(x)
        device_counts.copy_(_ints(turn))
        graph.replay()
        torch.cuda.synchronize()
        starts, cached, slots = s.want.append(turn, n, max_count=most)
        assert step["slots"].tolist() == slots and step["cached"].tolist() == cached
        s.expect(turn, starts, cached, *tokens, y)
        s.histories()
    s.pools()


@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 8, 1]])
def test_layers_share_a_step_on_two_streams_and_in_two_graphs(counts):
    """One plan, several layers: one after the other, at once on other streams, and captured apart from the plan."""
    rows, h, d = 3, 4, 64
    s = _prefix(h, d, False, [500, 9, 260])
    layers = [{name: x.clone() for name, x in s.cache.items()} for _ in range(5)]
    step = paged.append_tokens(s.t, _ints(counts), sum(counts), max_count=max(counts))
    q, k, v = (x.cuda() for x in s.tokens(sum(counts)))
    call = lambda cache: paged.paged_attention(cache, s.t, step, q, k, v)   # noqa: E731
    ys = [call(layers[0])]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for cache, stream in zip(layers[1:3], streams):
        with torch.cuda.stream(stream):
            ys.append(call(cache))
    graphs = []
    for cache in layers[3:]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ys.append(call(cache))
    torch.cuda.synchronize()
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for y, cache in zip(ys[1:], layers[1:]):
        assert torch.equal(y, ys[0])
        assert torch.equal(torch.nan_to_num(cache["selected"]), torch.nan_to_num(layers[0]["selected"]))


@pytest.mark.parametrize("counts", [[1, 1, 200, 1], [5, 1, 1, 8]])
def test_layers_of_a_step_from_two_threads(counts):
    """Calls of one step on one stream by several threads at once: as one after the other."""
    import threading

    s = _prefix(4, 64, False, [600, 500, 30, 640])
    n, layers = sum(counts), 24
    caches = [{name: x.clone() for name, x in s.cache.items()} for _ in range(layers + 1)]
    step = paged.append_tokens(s.t, _ints(counts), n, max_count=max(counts))
    q, k, v = (x.cuda() for x in s.tokens(n))
    want = paged.paged_attention(caches[layers], s.t, step, q, k, v)
    torch.cuda.synchronize()
    ys, start = [None] * layers, threading.Barrier(4)

    def work(first):
        start.wait()
        for i in range(first, layers, 4):
            ys[i] = paged.paged_attention(caches[i], s.t, step, q, k, v)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for y, cache in zip(ys, caches):
        assert torch.equal(y, want)
        for name in ("k", "v", "selected"):
            assert torch.equal(torch.nan_to_num(cache[name]), torch.nan_to_num(caches[layers][name]))


def test_the_same_step_gives_the_same_bits():
    s = _prefix(4, 64, False, [3000 % 600, 9, 600])
    saved = [{name: x.clone() for name, x in s.cache.items()} for _ in range(3)]
    step = paged.append_tokens(s.t, _ints([1, 28, 7]), 36)
    q, k, v = (x.cuda() for x in s.tokens(36))
    ys = [paged.paged_attention(cache, s.t, step, q, k, v) for cache in saved]
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])
    assert torch.equal(torch.nan_to_num(saved[0]["selected"]), torch.nan_to_num(saved[2]["selected"]))


# ---- copies ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,dim,page,per_head,rows", [(2, 64, 16, False, 4), (3, 128, 32, True, 9), (2, 64, 128, False, 40)])
def test_copied_rows_go_on_as_their_parents(heads, dim, page, per_head, rows):
    rng = random.Random(rows)
    s = Served(rows, heads, dim, page, -(-400 // page), rows * (-(-400 // page)), per_head, scale=0.5, seed=rows)
    s.step([rng.choice([0, 1, page, 100, 37]) for _ in range(rows)])
    for _ in range(3):
        parents = [rng.choice([r, rng.randint(0, rows - 1), rng.randint(0, 1), -1]) for r in range(rows)]
        moves = paged.reorder_rows(s.t, _ints(parents))
        paged.move_rows(s.cache, moves)
        s.want.reorder(parents)
        _same_tables(s.t, s.want)
        old = list(s.rows)
        got = s.cache["selected"].cpu()
        for r, p in enumerate(parents):
            s.rows[r] = old[p] if p >= 0 else (old[r][0][:0], old[r][1][:0], old[r][2][:, :0])
            n = s.rows[r][0].shape[0]
            for i, name in enumerate(("k", "v")):
                ids = s.want.blocks[r]
                if n:
                    now = s.cache[name][ids].permute(1, 0, 2, 3).reshape(heads, -1, dim)[:, :n].permute(1, 0, 2).cpu().float()
                    assert torch.equal(now, s.rows[r][i]), (r, name)
            assert not torch.isnan(got[r, :, :n]).any()
        counts = [rng.choice([0, 1, 20]) for _ in range(rows)]
        n = sum(counts)
        step = _append(s.t, s.want, counts, n)
        q, k, v = s.tokens(n)
        y = s.slot.attend_pages(q.cuda(), k.cuda(), v.cuda(), s.cache, s.t, step)
        s.expect(counts, step["query_start"].tolist(), step["cached"].tolist(), q, k, v, y)


def test_histories_behind_the_last_token_stay():
    t = paged.begin_tables(3, 30, 16, 8, 2)
    cache = paged.begin_pages(t, 64)
    paged.append_tokens(t, _ints([21, 3, 50]), 74)
    cache["selected"].copy_(torch.randn(cache["selected"].shape))
    was = cache["selected"].clone()
    paged.move_rows(cache, paged.reorder_rows(t, _ints([2, 0, 1])))
    for r, (p, n) in enumerate(((2, 50), (0, 21), (1, 3))):
        assert torch.equal(cache["selected"][r, :, :n], was[p, :, :n]) and torch.equal(cache["selected"][r, :, n:], was[r, :, n:])


_REFUSED_LAUNCH = """
#define _GNU_SOURCE
#include <dlfcn.h>
typedef struct { unsigned x, y, z; } dim3_t;
static int left = -1, failed = 0;             /* launches until one is refused */
void refuse_launch(int n) { left = n; failed = 0; }
int cudaLaunchKernel(const void* f, dim3_t g, dim3_t b, void** a, unsigned long smem, void* s) {
  if (left >= 0 && left-- == 0) return failed = 2;                       /* cudaErrorMemoryAllocation */
  return ((int (*)(const void*, dim3_t, dim3_t, void**, unsigned long, void*))dlsym(RTLD_NEXT, "cudaLaunchKernel"))(f, g, b, a, smem, s);
}
int cudaLaunchKernelExC(const void* c, const void* f, void** a) {
  if (left >= 0 && left-- == 0) return failed = 2;
  return ((int (*)(const void*, const void*, void**))dlsym(RTLD_NEXT, "cudaLaunchKernelExC"))(c, f, a);
}
int cudaGetLastError(void) {
  const int e = failed;
  failed = 0;
  return e ? e : ((int (*)(void))dlsym(RTLD_NEXT, "cudaGetLastError"))();
}
"""

_RETRIED_STEP = """
import ctypes, sys
import torch
from selective_attention_b200 import _lib, paged
shim = ctypes.CDLL(sys.argv[1])
g = torch.Generator("cpu").manual_seed(3)
ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
t = paged.begin_tables(3, 1200, 16, 400, 4)
cache = paged.begin_pages(t, 64, per_head=sys.argv[2] == "per_head")
tokens = lambda n: [torch.randn(n, 4, 64, generator=g).bfloat16().cuda() for _ in range(3)]
first = [300, 5, 40]
paged.paged_attention(cache, t, paged.append_tokens(t, ints(first), sum(first)), *tokens(sum(first)))
for counts in ([200, 1, 1], [1, 1, 1], [3, 1, 8], [3000, 1, 1]):
    total, most = sum(counts), max(counts)
    tables = {k: x.clone() for k, x in t.items() if torch.is_tensor(x)}

    def tried(call, unchanged):
        before, n = _lib.launch_count(), 0
        while True:
            shim.refuse_launch(n)
            try:
                out = call()
                shim.refuse_launch(-1)
                torch.cuda.synchronize()
                return out, n
            except _lib.LibraryError as e:
                shim.refuse_launch(-1)
                assert e.status == 5, e
                torch.cuda.synchronize()
                unchanged(n)
                n += 1

    def same_tables(n):
        assert all(torch.equal(t[k], x) for k, x in tables.items()), n

    step, launches = tried(lambda: paged.append_tokens(t, ints(counts), total, max_count=most), same_tables)
    assert launches == (2 if total > 2048 else 1), launches
    history, old = cache["selected"].clone(), step["cached"].tolist()

    def same_history(n):
        assert all(torch.equal(cache["selected"][r, :, :c], history[r, :, :c]) for r, c in enumerate(old)), n

    x = tokens(total)
    want = {k: v.clone() for k, v in cache.items()}
    y = paged.paged_attention(want, t, step, *x)
    got, launches = tried(lambda: paged.paged_attention(cache, t, step, *x), same_history)
    assert torch.equal(got, y) and torch.equal(cache["selected"], want["selected"]), counts
    few = most == 200 and sys.argv[2] == "shared"              # selection of few tiles scans them, too
    assert launches == (1 if most <= 8 else 4 if few else 5), launches
print("all tried")
"""


@pytest.mark.parametrize("selectors", ["shared", "per_head"])
def test_a_step_whose_call_fails_can_be_tried_again(selectors, tmp_path):
    """Whichever of its launches is refused (by a stand-in for the runtime's launch functions, in a process of its own), the
    tables and the histories are what they were, and the step counts once when it goes through."""
    import os
    import subprocess
    import sys

    source, shim = tmp_path / "refuse.c", tmp_path / "refuse.so"
    source.write_text(_REFUSED_LAUNCH)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(shim), str(source), "-ldl"])
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "selective-attention-study_b200")
    env = dict(os.environ, LD_PRELOAD=str(shim), PYTHONPATH=os.pathsep.join([package, os.environ.get("PYTHONPATH", "")]))
    run = subprocess.run([sys.executable, "-c", _RETRIED_STEP, str(shim), selectors], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all tried" in run.stdout, run.stdout + run.stderr
