"""Beam selection against its oracle in 64 bits, and a beam search over the paged cache against one that keeps whole sequences."""

import pytest
import torch

import paged_oracle
from selective_attention_b200 import beams, kernels, paged

pytestmark = pytest.mark.gpu


def _check(logits, scores, width):
    got, rows, tokens = (x.cpu() for x in beams.beam_select(logits, scores, width))
    want, want_rows, want_tokens = paged_oracle.select(logits.cpu(), scores.cpu(), width)
    assert rows.dtype == torch.int32 and tokens.dtype == torch.int64 and got.dtype == torch.float32
    assert torch.equal(rows.long(), want_rows) and torch.equal(tokens, want_tokens)
    # 32-bit exponentials in the sum (2^-21 of it each at most), the sum itself over a thread's 32 and the tree's 8, the output's rounding
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    fine = torch.isfinite(want)
    bound = 2.0 ** -24 * want.abs() + 2.0 ** -21 + 2.0 ** -24 * 64
    assert ((got.double() - want).abs() <= bound)[fine].all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,n,vocab,width", [(1, 1, 1, 1), (1, 1, 7, 5), (2, 3, 33, 32), (1, 4, 50257, 4), (3, 5, 8191, 11), (40, 8, 5003, 8),
                                                  (1, 1, 50304, 32), (2, 256, 300, 9), (70, 12, 2049, 32), (13, 2, 388, 5),
                                                  (13, 7, 244, 10), (3, 1, 257, 32), (2, 2, 2056, 31)])
def test_selection(dtype, groups, n, vocab, width):
    gen = torch.Generator().manual_seed(vocab + width)
    logits = (torch.randn(groups, n, vocab, generator=gen) * 3).to(dtype).cuda()
    scores = (-5 * torch.rand(groups, n, generator=gen)).cuda()
    _check(logits, scores, width)


def test_strided_and_unaligned_logits():
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(3, 9, 1003, generator=gen).bfloat16().cuda()
    scores = torch.randn(3, 9, generator=gen).cuda()
    _check(wide[:, 1:6, 3:], scores[:, 1:6], 7)
    _check(wide.transpose(0, 1)[2:5], scores.t()[2:5], 7)
    _check(wide[:, :, ::2], scores, 6)
    _check(wide[:1, :1].expand(2, 4, 1003), scores[:2, :4], 5)


def test_equal_and_masked_logits():
    scores = torch.tensor([[-1.0, -1.0, -3.0]]).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        _check(torch.zeros(1, 3, 40000, dtype=dtype).cuda(), scores, 32)                    # everything equal
        x = torch.full((1, 3, 40000), -float("inf"), dtype=dtype)
        x[0, 0, 39999], x[0, 1, 17], x[0, 2, 20000:20003] = 1.0, 2.0, 0.5                   # five that may be taken
        _check(x.cuda(), scores, 9)
        x = torch.randint(0, 3, (1, 3, 40000), generator=torch.Generator().manual_seed(2)).to(dtype)
        _check(x.cuda(), scores, 32)


def test_first_step_and_values_that_are_not_finite():
    gen = torch.Generator().manual_seed(4)
    inf, nan = float("inf"), float("nan")
    logits = torch.randn(5, 4, 3000, generator=gen)
    scores = torch.tensor([[0.0, -inf, -inf, -inf], [-1.0, -2.0, nan, -3.0], [0.0, 0.0, 0.0, 0.0], [-inf] * 4, [0.0, -1.0, -2.0, -inf]])
    logits[0, 1:] = logits[0, :1]
    logits[2, 0, 77], logits[2, 1, 5], logits[2, 2] = nan, inf, -inf
    logits[4, 0, 100:] = -inf
    logits[4, 0, :100] = 30000.0
    for width in (4, 32):
        _check(logits.cuda(), scores.cuda(), width)


@pytest.mark.parametrize("groups,n,vocab,width", [(1, 32, 50304, 32), (3, 16, 20011, 32), (2, 256, 9000, 32), (1, 256, 6000, 5), (2, 33, 300, 32),
                                                  (1, 5, 200000, 32)])
def test_many_candidates(groups, n, vocab, width):
    """Where a group has more candidates than its threads keep at hand: ordinary beams; then with masked, poor and equal ones among them."""
    gen = torch.Generator().manual_seed(n + width)
    logits = (torch.randn(groups, n, vocab, generator=gen) * 3).bfloat16()
    scores = -5 * torch.rand(groups, n, generator=gen)
    _check(logits.cuda(), scores.cuda(), width)
    scores[:, 1::3] = -float("inf")
    logits[:, 0, 7:], logits[:, 2::4] = -float("inf"), logits[:, :1, :1]
    logits[:, 3, vocab // 2], logits[:, 4, 1] = float("nan"), float("inf")
    _check(logits.cuda(), scores.cuda(), width)
    scores[:, 1:] = -float("inf")                                 # a search's first step
    _check(logits.cuda(), scores.cuda(), width)
    _check(torch.zeros_like(logits).cuda(), torch.zeros_like(scores).cuda(), width)
    logits = (torch.randn(groups, n, vocab, generator=gen) * 3).bfloat16()
    for far in (3.0, 100.0):                                      # one beam far above the others
        scores = -far - torch.rand(groups, n, generator=gen)
        scores[:, n // 2] = 0.0
        _check(logits.cuda(), scores.cuda(), width)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("warps", [3, 5, 6, 7])
@pytest.mark.parametrize("width", [29, 30, 31, 32])
def test_runs_whose_warps_do_not_divide_the_width(dtype, warps, width):
    """A run of 3, 5, 6 or 7 warps of 16-byte units: twice as many maxima a warp as an even share are more than 64 in all.  Drawn
    logits, and maxima gathered in two or three warps so that the last of the first `width` lies far down in one of them."""
    gen = torch.Generator().manual_seed(100 * warps + width)
    per = 4 if dtype == torch.float32 else 8
    for units in (32 * warps, 32 * warps - 31, 32 * warps - 9):
        logits = torch.randn(40, 1, units * per, generator=gen)
        scores = -torch.rand(40, 1, generator=gen)
        _check(logits.to(dtype).cuda(), scores.cuda(), width)
        _check(logits[:39].view(13, 3, units * per).to(dtype).cuda(), scores[:39].view(13, 3).cuda(), width)
        each = 2 * -(-width // warps)
        for g in range(40):
            # `each` high units in one warp, the lowest of them; as many in the next as reach maximum 63; the others wherever there is room
            order = [63 % warps] + [w for w in torch.randperm(warps, generator=gen).tolist() if w != 63 % warps]
            low = order.pop(1 + g % (warps - 1))
            room = [min(32, units - 32 * w) for w in order]
            left, takes = width - min(each, min(32, units - 32 * low)), []
            for w, n in zip(order, room):
                takes.append((w, min(left, n, 63 // warps + 1)))
                left -= takes[-1][1]
            value = 16.0 + 0.125 * width                          # downwards in steps that every type has
            for w, n in takes + [(low, width - sum(n for _, n in takes))]:
                for u in torch.randperm(min(32, units - 32 * w), generator=gen)[:n].tolist():
                    logits[g, 0, (32 * w + u) * per + (u + g) % per] = value
                    value -= 0.125
        _check(logits.to(dtype).cuda(), scores.cuda(), width)


@pytest.mark.parametrize("dtype,per", [(torch.float32, 4), (torch.bfloat16, 8)])
def test_a_long_vocabulary_with_a_short_last_run(dtype, per):
    """488 runs of 512 units and one of 160 (five warps), which holds the best."""
    gen = torch.Generator().manual_seed(per)
    vocab = (488 * 512 + 160) * per
    logits = torch.randn(1, 1, vocab, generator=gen)
    for _ in range(6):
        logits[0, 0, -160 * per:] = torch.randn(160 * per, generator=gen)
        for w, n in ((3, 13), (1, 5), (0, 14)):                   # the 14th of warp 0 is the last of 32
            units = torch.randperm(32, generator=gen)[:n] + 32 * w
            logits[0, 0, (488 * 512 + units) * per + 1] = 16.0 + 0.125 * torch.arange(n) + 4 * (w > 0) + 2 * (w > 1)
        _check(logits.to(dtype).cuda(), torch.zeros(1, 1).cuda(), 32)


def test_arguments_that_are_refused():
    x, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in ((x, s, 0), (x, s, 31), (x, s, 33), (x.long(), s, 2), (x, s.cpu(), 2), (x[:, :0], s[:, :0], 1), (x, s[:, :2], 2)):
        with pytest.raises(ValueError):
            beams.beam_select(*bad)


def test_a_captured_selection_is_replayed():
    x, s = torch.zeros(2, 4, 9001, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beams.beam_select(x, s, 6)
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        s.copy_(torch.randn(s.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = beams.beam_select(x, s, 6)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_beam_search_over_the_paged_cache():
    """Two prompts, four beams each, against a search whose beams are whole sequences, attended from the start in every step.  One
    layer; embeddings, projections and head are drawn."""
    gen = torch.Generator().manual_seed(11)
    vocab, h, d, n, steps, prompts = 97, 4, 64, 4, 24, (37, 80)
    table = torch.randn(vocab, 3, h, d, generator=gen).bfloat16().cuda()
    head = (torch.randn(h * d, vocab, generator=gen) * 0.2).cuda()
    rows = len(prompts) * n
    words = [torch.randint(0, vocab, (p,), generator=gen).tolist() for p in prompts]

    def whole(sequence):
        qkv = table[torch.tensor(sequence, device="cuda")]
        return kernels.selective_attention_forward(*(qkv[:, i].transpose(0, 1)[None] for i in range(3)))[0, :, -1].reshape(-1)

    t = paged.begin_tables(rows, 60, 16, 8, h)
    cache = paged.begin_pages(t, d)

    def feed(tokens, counts, most):
        step = paged.append_tokens(t, torch.tensor(counts, dtype=torch.int32).cuda(), sum(counts), max_count=most)
        qkv = table[tokens]
        y = paged.paged_attention(cache, t, step, qkv[:, 0], qkv[:, 1], qkv[:, 2])
        return y, step

    first = [p if i == 0 else 0 for p in prompts for i in range(n)]
    y, step = feed(torch.tensor(sum(words, [])).cuda(), first, max(prompts))
    y = y[(step["query_start"][1:].long() - 1).clamp_min(0)].float().reshape(rows, -1)
    scores = torch.tensor([[0.0] + [-float("inf")] * (n - 1)] * len(prompts)).cuda()
    sequences = [list(words[r // n]) for r in range(rows)]
    for _ in range(steps):
        scores, parents, tokens = beams.beam_select((y @ head).view(len(prompts), n, vocab), scores, n)
        moves = paged.reorder_rows(t, parents.reshape(-1))
        paged.move_rows(cache, moves)
        sequences = [sequences[p] + [w] for p, w in zip(parents.reshape(-1).tolist(), tokens.reshape(-1).tolist())]
        y, _ = feed(tokens.reshape(-1), [1] * rows, 1)
        y = y.float().reshape(rows, -1)
        for r in (0, 3, 5, 7):
            want = whole(sequences[r])
            # two bf16 forms of one number: each rounds its output (2^-8) and the probabilities before it
            torch.testing.assert_close(y[r], want.float(), atol=2.0 ** -5, rtol=2.0 ** -6)
    assert len({tuple(x) for x in sequences}) == rows
    refs = torch.zeros(60, dtype=torch.int32)
    for r, length in enumerate(t["lengths"].tolist()):
        assert length == len(sequences[r])
        for page in t["block_tables"][r, :-(-length // 16)].tolist():
            refs[page] += 1
    assert torch.equal(refs, t["page_refs"].cpu()) and int((refs == 0).sum()) == int(t["free_count"])


def test_a_captured_search_step_is_replayed():
    """Selection, reordering, moves, tables and attention of a step in one graph, against the same calls one by one."""
    gen = torch.Generator().manual_seed(12)
    vocab, h, d, n, groups = 211, 4, 64, 3, 2
    table = torch.randn(vocab, 3, h, d, generator=gen).bfloat16().cuda()
    head = (torch.randn(h * d, vocab, generator=gen) * 0.2).cuda()
    rows = n * groups

    class Search:
        def __init__(self):
            self.t = paged.begin_tables(rows, 80, 16, 10, h)
            self.cache = paged.begin_pages(self.t, d)
            counts = torch.tensor([30, 0, 0, 47, 0, 0], dtype=torch.int32).cuda()
            step = paged.append_tokens(self.t, counts, 77)
            qkv = table[torch.arange(77, device="cuda")]
            y = paged.paged_attention(self.cache, self.t, step, *(qkv[:, i] for i in range(3)))
            self.y = y[(step["query_start"][1:].long() - 1).clamp_min(0)].float().reshape(rows, -1)
            self.scores = torch.tensor([[0.0] + [-float("inf")] * (n - 1)] * groups).cuda()
            self.ones = torch.ones(rows, dtype=torch.int32).cuda()

        def step(self):
            scores, parents, tokens = beams.beam_select((self.y @ head).view(groups, n, vocab), self.scores, n)
            paged.move_rows(self.cache, paged.reorder_rows(self.t, parents.reshape(-1)))
            step = paged.append_tokens(self.t, self.ones, rows, max_count=1)
            qkv = table[tokens.reshape(-1)]
            y = paged.paged_attention(self.cache, self.t, step, *(qkv[:, i] for i in range(3)))
            self.scores.copy_(scores)
            self.y.copy_(y.float().reshape(rows, -1))
            return tokens, parents

    eager, captured = Search(), Search()
    want = [[x.clone() for x in eager.step()] for _ in range(20)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        warm = Search()
        warm.step()                                                # the library's set-up calls come before a capture
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured.step()
    for tokens, parents in want:
        graph.replay()
        assert torch.equal(out[0], tokens) and torch.equal(out[1], parents)
    assert torch.equal(captured.y, eager.y) and torch.equal(captured.scores, eager.scores)
    for name in ("block_tables", "lengths", "page_refs", "free_count"):
        assert torch.equal(captured.t[name], eager.t[name])
