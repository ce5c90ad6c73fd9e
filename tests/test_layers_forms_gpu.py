"""Layer norm, the embedding and the loss over a vocabulary where torch, a mask or a size asks something unusual of them."""

import pytest
import torch

from selective_attention_b200 import layers

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _calls():
    """Every call by itself: what it takes that may have a derivative, and the call of these."""
    x, branch, w = (torch.randn(4, 32, device="cuda") for _ in range(3))
    p, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    t = torch.tensor([0, 1, 2, 3], device="cuda")
    return {
        "layer_norm": ([x, p, b], layers.layer_norm), "add_layer_norm": ([x, branch, p, b], layers.add_layer_norm),
        "embedding": ([w], lambda a: layers.embedding(t, a)), "linear_cross_entropy": ([x, w], lambda a, c: layers.linear_cross_entropy(a, c, t)),
        "linear_cross_entropy of each": ([x, w], lambda a, c: layers.linear_cross_entropy(a, c, t, reduction="none")),
    }


@pytest.mark.parametrize("name", ["layer_norm", "add_layer_norm", "embedding", "linear_cross_entropy", "linear_cross_entropy of each"])
def test_tangents_and_batches_of_a_transform_are_refused(name):
    """Dropped, a tangent would read as a derivative of zero."""
    inputs, call = _calls()[name]
    want = call(*inputs)
    for i in range(len(inputs)):
        for wants in (False, True):
            args = [a.clone().requires_grad_(wants) for a in inputs]
            with torch.autograd.forward_ad.dual_level():
                args[i] = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
                again = call(*inputs)                       # others are taken as ever
                assert all(torch.equal(a, b) for a, b in zip(again if isinstance(again, tuple) else [again], want if isinstance(want, tuple) else [want]))
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda a: call(*inputs[:i], a, *inputs[i + 1:]), (inputs[i],), (torch.ones_like(inputs[i]),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda a: call(*inputs[:i], a, *inputs[i + 1:]))(inputs[i][None])


def _gradients(x, w, targets, reduction):
    a, b = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    loss = layers.linear_cross_entropy(a, b, targets, reduction=reduction)
    return [loss.detach(), *torch.autograd.grad(loss, (a, b), torch.ones_like(loss))]


@pytest.mark.parametrize("masked", [-1e4, -1e8, -3e8, -1e10, -1e30, -2e38])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_words_masked_by_any_number_leave_the_others_alone(dtype, masked):
    """A column of ones and a bias of the words in the table; whole tiles of nothing but masked words, before, between and behind others."""
    gen = torch.Generator("cpu").manual_seed(51)
    x, w = torch.randn(150, 64, generator=gen).to(dtype).cuda(), (torch.randn(1500, 64, generator=gen) * 0.2).to(dtype).cuda()
    kept = torch.zeros(1500, dtype=torch.bool, device="cuda")
    kept[520:700], kept[1100:1180] = True, True
    x[:, 63] = 1
    w[:, 63] = 0
    w[~kept] = 0
    w[~kept, 63] = masked
    words = kept.nonzero()[:, 0]
    at = torch.randint(0, len(words), (150,), generator=gen).cuda()
    for reduction in ("none", "sum"):
        loss, dx, dw = _gradients(x, w, words[at], reduction)
        want, wanted, dwant = _gradients(x, w[kept], at, reduction)
        assert torch.isfinite(loss).all() and (loss - want).abs().max() <= 2.0 ** -20 * (150 if reduction == "sum" else 1) * 8
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -20          # the same sums, of more or fewer tiles
        assert (dx.float() - wanted.float()).abs().max() <= 2 * half * wanted.float().abs().max()
        assert (dw[kept].float() - dwant.float()).abs().max() <= 2 * half * dwant.float().abs().max() and (dw[~kept] == 0).all()
    # rows that the mask leaves nothing of: all words alike
    loss, dx, _ = _gradients(x, w[~kept], at, "none")
    assert (loss - torch.log(torch.tensor(1500.0 - len(words)))).abs().max() < 2.0 ** -18 and torch.isfinite(dx).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [30.0, 1e3, 1e4, 1e6])
def test_logits_of_any_size(dtype, scale):
    """Up to 10^13: losses of nothing or of about as much, as their products are rounded."""
    gen = torch.Generator("cpu").manual_seed(52)
    x, w = ((torch.randn(n, 64, generator=gen) * scale).to(dtype).cuda() for n in (200, 900))
    z = x.double() @ w.double().T
    targets = z.argmax(1)
    targets[::2] = torch.randint(0, 900, (100,), generator=gen).cuda()
    p = torch.softmax(z, 1)
    off = 18 * 2.0 ** -22 * (x.double().abs() @ w.double().abs().T).amax(1)          # of any logit: 64 / 16 groups of products, in up to 3 parts
    want = torch.logsumexp(z, 1) - z.gather(1, targets[:, None])[:, 0]
    loss, dx, dw = _gradients(x, w, targets, "none")
    assert ((loss.double() - want).abs() <= 2 * off + 2.0 ** -20 * (1 + want)).all()
    # half the targets are the largest word by far: nothing is left of their gradients
    sure = (1 - p.gather(1, targets[:, None])[:, 0] < 1e-30) & (z.topk(2).values.diff(dim=1)[:, 0].abs() > 4 * off + 100)
    # but for exp2(r) of a rounding r of the largest logit times log2 e, of up to 8: 2^-22 of itself, its logarithm 2^-24 of up to 8 and as
    # much again for r taken from it, so 2^-20 in the loss, and in dz, whose exponential adds 2^-22
    assert sure.sum() > 60 and (loss[sure].abs() < 2.0 ** -20).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    assert (dx[sure].abs() <= 2.0 ** -19 * w.float().abs().amax()).all()
    import test_layers_gpu

    total, dx, dw = test_layers_gpu._with_the_loss(x, w, targets, -100, "sum", dtype, torch.ones((), device="cuda"))
    assert abs(float(total) - float(want.sum())) <= float((2 * off + 2.0 ** -20 * (1 + want)).sum()) + 2.0 ** -23 * float(want.sum())
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and (dx[sure] == 0).all()


def _definition(x, w, targets):
    """Losses, and the gradients of their sum, in 64 bits."""
    x, w = x.double(), w.double()
    z = x @ w.T
    lse = torch.logsumexp(z, 1, keepdim=True)
    losses = (lse - z.gather(1, targets[:, None]))[:, 0]
    dz = torch.exp_(z.sub_(lse)).scatter_add_(1, targets[:, None], -torch.ones_like(lse))
    return losses, dz @ w, dz.T @ x


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype,bound", [(BF16, 1e-6), (F16, 1e-6), (F32, 6e-7)])
@pytest.mark.parametrize("tokens", [100, 300])
@pytest.mark.parametrize("width", [2048, 4096, 16384])
def test_a_wide_products_error_does_not_grow_with_its_width(width, tokens, dtype, bound):
    """A group of 16 products loses up to 2^-23 of what is summed so far, towards zero: half of that over 512 of the contraction, on what
    is half of its sum on average, is 5e-7 of the sum (of 256, 2.4e-7); several such sums have signs of their own.  Over the whole width,
    the loss was 1.4e-6, 2.8e-6 and 1.1e-5 off; fp32 gradients 1.7e-6, 3.4e-6 and 1.2e-5."""
    gen = torch.Generator("cuda").manual_seed(61)
    x = torch.randn(tokens, width, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(3000, width, generator=gen, device="cuda") * 3.0 / width ** 0.5).to(dtype)
    targets = torch.randint(0, 3000, (tokens,), generator=gen, device="cuda")
    losses, dx, dw = _definition(x, w, targets)
    got = _gradients(x, w, targets, "none")
    with torch.no_grad():
        alone = layers.linear_cross_entropy(x, w, targets, reduction="none")
    assert _off(got[0], losses) < bound and _off(alone, losses) < bound
    # e^z has z's error times its size, of 3 to 10 here, beside roundings to the type
    half = torch.finfo(dtype).eps / 2
    grads = [got[1:]]
    if dtype != F16:
        import test_layers_gpu

        total, *with_the_loss = test_layers_gpu._with_the_loss(x, w, targets, -100, "sum", dtype, torch.ones((), device="cuda"))
        assert abs(float(total) - float(losses.sum())) < bound * float(losses.sum())
        grads.append(with_the_loss)
    for a, b in grads:
        assert _off(a, dx) < 1.2e-6 + half and _off(b, dw) < 1.2e-6 + half


@pytest.mark.parametrize("tokens,vocab,width", [(8000, 600, 72), (70, 60000, 40), (4000, 9000, 520)])
def test_a_long_sums_error_in_fp32_does_not_grow_with_its_length(tokens, vocab, width):
    """Sums of the gradients over tokens and words: 2.4e-6 where 2,048 of the contraction were added towards zero."""
    gen = torch.Generator("cuda").manual_seed(62)
    x, w = (torch.randn(n, width, generator=gen, device="cuda") for n in (tokens, vocab))
    w *= 3.0 / width ** 0.5
    targets = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    losses, dx, dw = _definition(x, w, targets)
    import test_layers_gpu

    ones = torch.ones((), device="cuda")
    for loss, a, b in (_gradients(x, w, targets, "none"), test_layers_gpu._with_the_loss(x, w, targets, -100, "sum", F32, ones)):
        assert _off(loss, losses if loss.dim() else losses.sum()) < 6e-7 and _off(a, dx) < 1.2e-6 and _off(b, dw) < 1.2e-6


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_what_rows_of_a_table_have_in_common_keeps_its_size(reduction):
    """dx is a mean of the table's rows less one of them; the rows' own mean of 1 enters and leaves.  Towards zero, 50,304 words lost 2.9e-4
    of it, 1.8 times what dx is rounded by."""
    gen = torch.Generator("cuda").manual_seed(63)
    x = (torch.randn(4864, 1024, generator=gen, device="cuda") * 0.2).to(BF16)
    w = (1 + torch.randn(50304, 1024, generator=gen, device="cuda") * 0.1).to(BF16)
    targets = torch.randint(0, 50304, (4864,), generator=gen, device="cuda")
    a = x.clone().requires_grad_(True)
    loss = layers.linear_cross_entropy(a, w, targets, reduction=reduction)
    (dx,) = torch.autograd.grad(loss, a, torch.ones_like(loss))
    _, want, _ = _definition(x[:64], w, targets[:64])
    # 8,192 words are 512 groups of 2^-23 at most; roundings of dx and of the exponentials have no sign
    assert abs(float((dx[:64].double() - want).mean())) < 512 * 2.0 ** -23 + 2e-5
    assert _off(dx[:64], want) < 0.55 * 2.0 ** -8                 # a rounding to 8 bits is 0.43 of its half step in the norm


@pytest.mark.parametrize("dtype,tokens,vocab,width,reduction", [
    (BF16, 41100, 4500, 72, "none"), (F16, 50000, 4200, 40, "mean"), (F32, 15000, 5000, 65, "none"), (F16, 90001, 2500, 261, "none"),
    (F32, 40000, 1500, 20, "sum"), (BF16, 600000, 260, 24, "mean"), (BF16, 130000, 5000, 8, "none")])
def test_more_tokens_than_a_run_of_the_gradients(dtype, tokens, vocab, width, reduction):
    """Runs of tokens, and in them pieces of the vocabulary, ragged both: 320 MB of what stands for logits at a time."""
    gen = torch.Generator("cuda").manual_seed(71)
    x = torch.randn(tokens, width, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(vocab, width, generator=gen, device="cuda") * 2.0 / width ** 0.5).to(dtype)
    targets = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    targets[3::7] = -100
    targets[tokens // 2:tokens // 2 + 2000] = -100
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    g = torch.rand(tokens, generator=gen, device="cuda") + 0.5 if reduction == "none" else torch.tensor(0.75 if dtype != F16 else 768.0, device="cuda")
    loss = layers.linear_cross_entropy(a, b, targets, reduction=reduction)
    got = torch.autograd.grad(loss, (a, b), g, retain_graph=True)
    again = torch.autograd.grad(loss, (a, b), g)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    counts = targets != -100
    each = torch.where(counts, g.double(), 0.0) / (int(counts.sum()) if reduction == "mean" else 1)
    dx, dw, losses = torch.empty(tokens, width, dtype=torch.float64, device="cuda"), torch.zeros(vocab, width, dtype=torch.float64, device="cuda"), []
    for i in range(0, tokens, 10000):
        rows = slice(i, i + 10000)
        z = x[rows].double() @ w.double().T
        logp, at = torch.log_softmax(z, 1), targets[rows].clamp(min=0)[:, None]
        losses.append(torch.where(counts[rows], -logp.gather(1, at)[:, 0], 0.0))
        dz = logp.exp_().scatter_add_(1, at, -torch.ones(len(at), 1, dtype=torch.float64, device="cuda")) * each[rows, None]
        dx[rows] = dz @ w.double()
        dw += dz.T @ x[rows].double()
    losses = torch.cat(losses)
    want = losses if reduction == "none" else losses.sum() / (int(counts.sum()) if reduction == "mean" else 1)
    assert _off(loss.detach(), want) < 6e-7
    # dx: its rounding and, of 16 bits, that of what is not at the target; dw: its rounding and dz's
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 1.2e-6
    assert _off(got[0], dx) < 0.55 * half + 1.2e-6 and _off(got[1], dw) < 0.66 * half + 1.2e-6 and (got[0][~counts] == 0).all()
    one = torch.autograd.grad(layers.linear_cross_entropy(a, b.detach(), targets, reduction=reduction), a, g)[0]
    other = torch.autograd.grad(layers.linear_cross_entropy(a.detach(), b, targets, reduction=reduction), b, g)[0]
    assert torch.equal(one, got[0]) and torch.equal(other, got[1])


def test_a_far_row_has_its_own_run_alone_gone_through_once_more():
    """Eight runs of tokens; the product of the logits is about a quarter of a run."""
    import test_layers_gpu

    gen = torch.Generator("cuda").manual_seed(81)
    x = torch.randn(16384, 512, generator=gen, device="cuda").to(BF16)
    w = (torch.randn(131072, 512, generator=gen, device="cuda") * 0.05).to(BF16)
    targets = torch.randint(0, 131072, (16384,), generator=gen, device="cuda")
    ones, far = torch.ones((), device="cuda"), x.clone()
    far[7] = w[(targets[7] + 1) % 131072] * 200             # the logit of another word is 256
    times = {}
    for _ in range(4):
        for name, a in (("near", x), ("far", far)):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            loss, dx, _ = test_layers_gpu._with_the_loss(a, w, targets, -100, "sum", BF16, ones)
            end.record()
            torch.cuda.synchronize()
            times[name] = min(times.get(name, 1e9), begin.elapsed_time(end))
            assert torch.isfinite(loss) and torch.isfinite(dx).all()
    assert times["far"] < 1.13 * times["near"], times       # 1.03; with every later run once more 1.25


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,reduction", [(1, "sum"), (2, "none"), (9, "mean"), (64, "none"), (128, "sum")])
def test_few_tokens_dw_is_as_exact_as_its_type(tokens, reduction, dtype):
    """dz in two parts; in one, a token's whole part of dw would be off by what its target's dz is rounded by."""
    for seed in range(6):
        gen = torch.Generator("cuda").manual_seed(90 + seed)
        x = torch.randn(tokens, 1000, generator=gen, device="cuda").to(dtype)
        w = (torch.randn(300, 1000, generator=gen, device="cuda") * 0.1).to(dtype).requires_grad_(True)
        targets = torch.randint(0, 300, (tokens,), generator=gen, device="cuda")
        loss = layers.linear_cross_entropy(x, w, targets, reduction=reduction)
        g = (torch.rand(loss.shape, generator=gen, device="cuda") + 0.5) * (1024.0 if dtype == F16 else 1.0)
        (dw,) = torch.autograd.grad(loss, w, g)
        z = x.double() @ w.detach().double().T
        dz = torch.softmax(z, 1) - torch.nn.functional.one_hot(targets, 300)
        want = (dz * (g if reduction == "none" else g / (tokens if reduction == "mean" else 1)).double().reshape(-1, 1)).T @ x.double()
        # a rounding to nearest is 0.43 of its half step in the norm, where values lie anywhere between two powers of two; of 1,000 that are
        # most of it, give or take a tenth
        assert _off(dw, want) < 0.48 * torch.finfo(dtype).eps / 2, seed


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_tokens_than_a_run_of_half_tiles(dtype):
    """Of 130,000 words 41,216 tokens' at a time: a token's loss is the same wherever it stands."""
    gen = torch.Generator("cuda").manual_seed(101)
    x = torch.randn(45000, 24, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(130000, 24, generator=gen, device="cuda") * 0.4).to(dtype)
    targets = torch.randint(0, 130000, (45000,), generator=gen, device="cuda")
    targets[41000:41500] = -100
    losses = layers.linear_cross_entropy(x, w, targets, reduction="none")
    halves = [layers.linear_cross_entropy(x[s], w, targets[s], reduction="none") for s in (slice(0, 20000), slice(20000, 45000))]
    assert torch.equal(losses, torch.cat(halves)) and (losses[41000:41500] == 0).all() and torch.isfinite(losses).all()
    for reduction in ("sum", "mean"):
        want = losses.double().sum() / (44500 if reduction == "mean" else 1)
        assert abs(float(layers.linear_cross_entropy(x, w, targets, reduction=reduction)) - float(want)) < 2.0 ** -22 * float(want)


def test_captured_gradients_of_several_runs_follow_their_inputs():
    gen = torch.Generator("cuda").manual_seed(102)
    x = torch.randn(41100, 40, generator=gen, device="cuda").to(BF16).requires_grad_(True)
    w = (torch.randn(4400, 40, generator=gen, device="cuda") * 0.3).to(BF16).requires_grad_(True)
    targets, g = torch.randint(0, 4400, (41100,), generator=gen, device="cuda"), torch.rand(41100, generator=gen, device="cuda")

    def step():
        return torch.autograd.grad(layers.linear_cross_entropy(x, w, targets, reduction="none"), (x, w), g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.mul_(0.5)
        w.neg_()
        targets[::3] = -100
        g.add_(0.25)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step())) and (got[0][::3] == 0).all()
