"""Layer norm, the embedding and the loss over a vocabulary against their definitions in 64 bits.

Tolerances count roundings: half a step of the result's type relative to the value, and steps of 2^-24 (2^-22 for a group of 16 products
that a tensor core adds, which truncates) relative to the sum of the magnitudes that were added."""

import ctypes
import math

import pytest
import torch

from selective_attention_b200 import _lib, layers

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _randn(gen, *shape, dtype=F32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float64) * scale + mean).to(dtype).cuda()


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check(name, got, want, slack):
    """got within half a step of its type and `slack` (broadcast) of the 64-bit value; subnormals of fp16 within their step."""
    assert got.shape == want.shape and torch.isfinite(want).all()
    off = (got.double() - want).abs()
    allowed = _half_step(got.dtype) * (want.abs() + slack) + slack + torch.finfo(got.dtype).smallest_normal
    assert torch.isfinite(got).all() and (off <= allowed).all(), (name, float((off / allowed).max()), float(off.max()))


# ---- layer norm -----------------------------------------------------------------------------------------------------------------

def _norm_reference(s, weight, bias, eps):
    mean = s.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((s - mean).square().mean(-1, keepdim=True) + eps)
    h = (s - mean) * r
    w = torch.ones(s.shape[-1], dtype=torch.float64, device="cuda") if weight is None else weight.double()
    y = h * w + (0.0 if bias is None else bias.double())
    return h, r, w, y


NORMS = [
    # shape, x, branch, weight, y, bias
    ((1, 1), F32, None, F32, F32, True), ((3, 7), BF16, None, BF16, BF16, False), ((2, 5, 64), F16, None, F16, F16, True),
    ((33, 200), BF16, BF16, BF16, BF16, False), ((9, 256), F32, BF16, F32, BF16, True), ((17, 257), F32, F16, F32, F16, True),
    ((130, 512), F32, F32, F32, F32, False), ((5, 513), BF16, None, F32, F32, True), ((2100, 768), BF16, None, BF16, BF16, True),
    ((70, 1024), F32, BF16, F32, BF16, False), ((66, 1025), F16, F16, F16, F16, True), ((31, 2048), BF16, F32, F32, BF16, False),
    ((6, 3000), F32, None, F32, BF16, True), ((5, 8192), F32, None, F32, F32, True), ((3, 8193), BF16, None, BF16, BF16, False),
    ((4, 16384), F32, BF16, F32, BF16, True),
]


@pytest.mark.parametrize("shape,xt,bt,wt,yt,bias", NORMS)
def test_layer_norm_and_its_gradients(shape, xt, bt, wt, yt, bias):
    gen, eps, width = _gen(sum(shape)), 1e-5, shape[-1]
    x = _randn(gen, *shape, dtype=xt, scale=2.0, mean=0.5).requires_grad_(True)
    branch = None if bt is None else _randn(gen, *shape, dtype=bt).requires_grad_(True)
    weight = _randn(gen, width, dtype=wt, scale=0.3, mean=1.0).requires_grad_(True)
    b = _randn(gen, width, dtype=wt).requires_grad_(True) if bias else None
    dy, dsum = _randn(gen, *shape, dtype=yt), _randn(gen, *shape, dtype=xt)
    if branch is None:
        y, leaves = layers.layer_norm(x, weight, b, eps=eps, dtype=yt), [x, weight] + ([b] if bias else [])
        grads = torch.autograd.grad(y, leaves, dy)
        s = x.detach().double()
        dsum64 = 0.0
    else:
        summed, y = layers.add_layer_norm(x, branch, weight, b, eps=eps, dtype=yt)
        leaves = [x, branch, weight] + ([b] if bias else [])
        grads = torch.autograd.grad([summed, y], leaves, [dsum, dy])
        want = x.detach().double() + branch.detach().double()
        _check("sum", summed.detach(), want, want.abs() * 2.0 ** -24)
        s, dsum64 = summed.detach().double(), dsum.double()
    assert y.dtype == yt and [g.dtype for g in grads] == [t.dtype for t in leaves]
    h, r, w, want = _norm_reference(s, weight.detach(), None if b is None else b.detach(), eps)
    step = 2.0 ** -24
    # the mean and the variance are sums of 16 values a thread and a tree: 32 steps of the largest value each
    slack = 64 * step * (s.abs().amax(-1, keepdim=True) * r + h.abs()) * w.abs() + step * (0.0 if b is None else b.detach().double().abs())
    _check("y", y.detach(), want, slack)
    g = dy.double() * w
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    want = r * (g - m1 - h * m2) + dsum64
    off_h = 64 * step * (s.abs().amax(-1, keepdim=True) * r + h.abs())
    most = g.abs().amax(-1, keepdim=True)
    slack = r * (64 * step * (most + h.abs() * most * h.abs().amax(-1, keepdim=True)) + off_h * most * (1 + 2 * h.abs().amax(-1, keepdim=True)))
    slack = slack + step * (want.abs() + (0.0 if branch is None else dsum64.abs()))
    _check("dx", grads[0], want, slack)
    if branch is not None:
        _check("dbranch", grads[1], want, slack)
    rows = tuple(range(len(shape) - 1))
    many = 256                                      # rows a CTA adds up, and its parts
    at = 1 if branch is None else 2
    _check("dweight", grads[at], (dy.double() * h).sum(rows), (many * step * (dy.double() * h).abs() + dy.double().abs() * off_h).sum(rows))
    if bias:
        _check("dbias", grads[at + 1], dy.double().sum(rows), many * step * dy.double().abs().sum(rows))


@pytest.mark.parametrize("shape,xt,bt,yt,bias", [
    ((1, 5), F32, None, F32, True), ((50001, 3), BF16, None, BF16, True), ((9999, 7), F32, BF16, BF16, True), ((257, 1), F32, None, BF16, True),
    ((5000, 8), BF16, BF16, BF16, False), ((129, 8), F32, None, F32, True), ((4097, 9), F16, F16, F16, True), ((3, 700, 16), BF16, None, F32, False),
    ((2049, 15), F16, None, F32, True), ((63, 31), F32, F16, F32, True), ((30011, 32), BF16, BF16, BF16, True), ((2, 24), F16, None, F16, False)])
def test_rows_of_a_few_values(shape, xt, bt, yt, bias):
    """One, two or four threads a row."""
    test_layer_norm_and_its_gradients(shape, xt, bt, F32 if xt == F32 else xt, yt, bias)


@pytest.mark.parametrize("shape,xt,bt,yt,bias", [
    ((700, 8192), BF16, None, BF16, True), ((451, 8200), F16, None, F16, False), ((601, 12288), BF16, BF16, BF16, True), ((333, 16384), F32, None, F32, True),
    ((449, 8191), F32, BF16, BF16, True), ((901, 4097), F16, None, F32, True), ((750, 4096), F32, BF16, F32, False)])
def test_rows_of_many_values(shape, xt, bt, yt, bias):
    """Several rows a CTA, whose columns' sums are in registers or in shared memory."""
    test_layer_norm_and_its_gradients(shape, xt, bt, F32 if xt == F32 else xt, yt, bias)


def test_layer_norm_without_parameters_and_without_gradients():
    gen = _gen(1)
    x = _randn(gen, 12, 100, dtype=BF16)
    y = layers.layer_norm(x)
    assert y.dtype == BF16 and not y.requires_grad
    assert torch.equal(y, layers.layer_norm(x.requires_grad_(True)).detach())
    ones, none = torch.ones(100, device="cuda", dtype=BF16), torch.zeros(100, device="cuda", dtype=BF16)
    assert torch.equal(y, layers.layer_norm(x.detach(), ones, none))
    only = layers.layer_norm(x.detach(), None, none.requires_grad_(True))
    assert torch.equal(only.detach(), y)
    only.sum().backward()
    assert (none.grad == 12).all()


def test_layer_norm_of_strided_rows_equals_that_of_their_copies():
    gen = _gen(2)
    base = _randn(gen, 6, 40, 3 * 96, dtype=F32)
    for x in (base[:, 3:30, 96:192], base[:, :, 1:98], base.transpose(1, 2), base[:1].expand(4, -1, -1), base[:, ::2]):
        w = _randn(gen, x.shape[-1]).requires_grad_(True)
        a, b = x.detach().requires_grad_(True), x.contiguous().detach().requires_grad_(True)
        ya, yb = layers.layer_norm(a, w), layers.layer_norm(b, w)
        assert torch.equal(ya, yb)
        dy = _randn(gen, *x.shape[:-1], 2 * x.shape[-1])[..., ::2]                   # a cotangent with strides of its own
        for p, q in zip(torch.autograd.grad(ya, (a, w), dy), torch.autograd.grad(yb, (b, w), dy.contiguous())):
            assert (p - q).abs().max() <= 2.0 ** -18 * q.abs().max()                 # 16-byte loads or not: another order of the sums
    y = layers.layer_norm(base[0, 0], w[:0].new_ones(288))
    assert y.shape == (288,)
    a = base[0].detach().requires_grad_(True)
    layers.layer_norm(a).sum().backward()                                            # a cotangent of stride 0
    assert a.grad.abs().max() < 1e-4


def test_layer_norm_of_no_rows_of_constant_rows_and_of_rows_that_are_not_finite():
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = layers.layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and (w.grad == 0).all()
    same = torch.full((3, 1024), 1000.0, device="cuda")
    assert (layers.layer_norm(same) == 0).all()
    rows = torch.randn(4, 64, device="cuda")
    rows[1, 5], rows[2, 7] = float("inf"), float("nan")
    y = layers.layer_norm(rows)
    assert torch.isnan(y[1]).any() and torch.isnan(y[2]).all()
    assert torch.equal(y[[0, 3]], layers.layer_norm(rows[[0, 3]]))


def test_only_one_of_the_two_results_of_add_layer_norm_is_used():
    gen = _gen(3)
    x, b = (_randn(gen, 50, 300).requires_grad_(True) for _ in range(2))
    w = _randn(gen, 300).requires_grad_(True)
    summed, y = layers.add_layer_norm(x, b, w)
    dy = _randn(gen, 50, 300)
    gx, gb, gw = torch.autograd.grad(y, (x, b, w), dy, retain_graph=True)
    s = summed.detach().requires_grad_(True)
    want = torch.autograd.grad(layers.layer_norm(s, w), (s, w), dy)
    assert torch.equal(gx, want[0]) and torch.equal(gb, want[0]) and torch.equal(gw, want[1])
    gx, gw = torch.autograd.grad(summed, (x, w), dy, allow_unused=True)
    assert torch.equal(gx, dy) and (gw is None or (gw == 0).all())


# ---- embedding -------------------------------------------------------------------------------------------------------------------

EMBEDDINGS = [
    # tokens, vocab, width, weight, y, skew
    (1, 1, 1, F32, F32, 0), (7, 3, 8, BF16, BF16, 0), (300, 50304, 768, BF16, BF16, 1), (31, 1, 64, F32, F32, 0), (32, 1, 64, F32, F32, 0),
    (33, 1, 64, F16, F16, 0), (1000, 2, 130, F32, BF16, 1), (5000, 257, 520, BF16, BF16, 1), (4097, 20000, 96, F32, F32, 1),
    (2000, 10, 3000, F32, F32, 2), (70, 5, 4104, BF16, BF16, 0), (20000, 300, 33, F16, F16, 1), (3000, 300000, 24, F32, F32, 0),
]


def _words(gen, tokens, vocab, skew):
    if skew == 0:
        return torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    upto = torch.cumsum(torch.arange(1, vocab + 1, dtype=torch.float64) ** -skew, 0)
    at = torch.searchsorted(upto, torch.rand(tokens, generator=gen, dtype=torch.float64) * upto[-1]).clamp(max=vocab - 1)
    return torch.randperm(vocab, generator=gen)[at].cuda()


@pytest.mark.parametrize("tokens,vocab,width,wt,yt,skew", EMBEDDINGS)
def test_embedding_and_its_gradient(tokens, vocab, width, wt, yt, skew):
    gen = _gen(tokens + vocab)
    idx = _words(gen, tokens, vocab, skew)
    weight = _randn(gen, vocab, width, dtype=wt).requires_grad_(True)
    scale = 1.7
    y = layers.embedding(idx, weight, scale=scale, dtype=yt)
    want = weight.detach().double()[idx] * torch.tensor(scale, dtype=F32).double().cuda()
    assert y.dtype == yt
    _check("y", y.detach(), want, want.abs() * 2.0 ** -24)
    dy = _randn(gen, tokens, width, dtype=yt)
    (dw,) = torch.autograd.grad(y, weight, dy)
    sums, sizes = (torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, idx, t) for t in (dy.double(), dy.double().abs()))
    count = torch.bincount(idx, minlength=vocab)[:, None].clamp(max=64 + tokens // 32)     # 32 tokens a piece, then the pieces
    assert dw.dtype == wt
    _check("dw", dw, sums * torch.tensor(scale, dtype=F32).double().cuda(), (count + 1) * 2.0 ** -24 * sizes * scale)
    (again,) = torch.autograd.grad(layers.embedding(idx, weight, scale=scale, dtype=yt), weight, dy)
    assert torch.equal(dw, again)                          # in an order of their own
    assert (dw[torch.bincount(idx, minlength=vocab) == 0] == 0).all()


def test_embedding_indices_outside_the_table_strides_and_shapes():
    gen = _gen(5)
    table = _randn(gen, 40, 3 * 32, dtype=BF16)
    weight = table[:, 32:64].detach().requires_grad_(True)
    idx = torch.tensor([[3, -1, 39], [40, 3, 1 << 40]], device="cuda")
    y = layers.embedding(idx, weight)
    assert y.shape == (2, 3, 32)
    bad = (idx < 0) | (idx >= 40)
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad].detach(), weight.detach()[idx[~bad]])
    dy = _randn(gen, 2, 3, 64, dtype=BF16)[..., ::2]
    (dw,) = torch.autograd.grad(y, weight, dy)
    want = torch.zeros(40, 32, dtype=torch.float64, device="cuda").index_add_(0, idx[~bad], dy[~bad].double())
    _check("dw", dw, want, want.abs() * 2.0 ** -22)
    assert torch.equal(layers.embedding(idx[0, :1].int(), weight), y[0, :1])
    none = layers.embedding(idx[:0], weight)
    assert none.shape == (0, 3, 32)
    none.sum().backward()
    assert (weight.grad == 0).all()
    y = layers.embedding(idx[0, [0, 2]], weight)                                    # all tokens outside but two
    y.sum().backward()
    assert weight.grad.sum() == 64


# ---- loss ------------------------------------------------------------------------------------------------------------------------

def _loss_reference(x, w, targets, ignore, g):
    """Losses, lse, dz, and the sums that bound the roundings, for cotangents g of the single losses."""
    x, w = x.detach().double(), w.detach().double()
    z = x @ w.T
    lse = torch.logsumexp(z, 1)
    counts = targets != ignore
    at = torch.where(counts, targets, 0)[:, None]
    losses = torch.where(counts, lse - z.gather(1, at)[:, 0], 0.0)
    dz = torch.exp(z - lse[:, None]).scatter_add_(1, at, -torch.ones_like(z[:, :1])) * torch.where(counts, g, 0.0)[:, None]
    return losses, dz, x.abs() @ w.abs().T


CODES = {F32: _lib.DTYPE_F32, BF16: _lib.DTYPE_BF16, F16: _lib.DTYPE_F16}


def _loss_struct(x, w, targets, ignore, reduction, product):
    p = _lib.LinearLoss()
    p.struct_bytes, p.product, p.x_dtype, p.weight_dtype = ctypes.sizeof(p), CODES[product], CODES[x.dtype], CODES[w.dtype]
    p.reduction, p.tokens, p.vocab, p.width = layers.REDUCTIONS[reduction], x.shape[0], w.shape[0], x.shape[1]
    p.ignore_index, p.x, p.x_stride, p.weight, p.weight_stride = ignore, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0)
    p.targets, p.stream = targets.data_ptr(), torch.cuda.current_stream().cuda_stream
    return p


def _with_the_loss(x, w, targets, ignore, reduction, product, dloss):
    """Loss and gradients by sa_linear_loss_train and _scale, which the Python call takes where they are the faster way."""
    lib, x, w, targets = _lib.load(), x.detach().reshape(-1, x.shape[-1]), w.detach(), targets.reshape(-1)
    p = _loss_struct(x, w, targets, ignore, reduction, product)
    loss, count = torch.empty((), device="cuda"), torch.empty(1, device="cuda")
    sums = [torch.full(t.shape, float("nan"), device="cuda") for t in (x, w)]
    p.loss, p.count, p.dx_sums, p.dweight_sums = (t.data_ptr() for t in (loss, count, *sums))
    p.workspace_bytes = lib.sa_linear_loss_train_bytes(ctypes.byref(p))
    workspace = torch.full((p.workspace_bytes,), 255, dtype=torch.uint8, device="cuda")
    p.workspace = workspace.data_ptr()
    _lib.check("sa_linear_loss_train", lib.sa_linear_loss_train(ctypes.byref(p)))
    dx, dw = torch.empty_like(x, memory_format=torch.contiguous_format), torch.empty_like(w, memory_format=torch.contiguous_format)
    p.dloss, p.dx, p.dweight = dloss.data_ptr(), dx.data_ptr(), dw.data_ptr()
    _lib.check("sa_linear_loss_scale", lib.sa_linear_loss_scale(ctypes.byref(p)))
    return loss, dx, dw


def _prefers(x, w, targets, ignore, reduction, product):
    x = x.detach().reshape(-1, x.shape[-1])
    return bool(_lib.load().sa_linear_loss_prefers_train(ctypes.byref(_loss_struct(x, w, targets, ignore, reduction, product))))


def _check_loss(x, w, targets, reduction, ignore=-100, product=None, seed=0, train=False):
    """``train``: by the C entries that compute the gradients with the loss."""
    gen = _gen(seed)
    n, (vocab, width) = targets.numel(), w.shape
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    product = product or x.dtype
    counts = int((targets != ignore).sum())
    if reduction == "none":
        dloss = (torch.rand(targets.shape, generator=gen) + 0.25).cuda()
        g = dloss.flatten().double()
    else:
        dloss = torch.tensor(0.75 if product != F16 else 768.0, device="cuda")
        g = dloss.double().expand(n) / (counts if reduction == "mean" else 1)
    if train:
        loss, dx, dw = _with_the_loss(x, w, targets, ignore, reduction, product, dloss)
        dx = dx.view(x.shape)
    else:
        train = _prefers(x, w, targets, ignore, reduction, product)
        loss = layers.linear_cross_entropy(x, w, targets, ignore_index=ignore, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), dloss)
    assert loss.dtype == F32 and (dx.dtype, dw.dtype, dx.shape, dw.shape) == (x.dtype, w.dtype, x.shape, w.shape)
    rx, rw = x.reshape(-1, width).to(product), w.to(product)
    losses, dz, sizes = _loss_reference(rx, rw, targets.flatten(), ignore, g)
    # a logit: width / 16 groups of products (in 3 parts: 6 times as many, of which the dropped ones are 2^-22), each truncated
    groups = -(-width // 64) * 4
    off = ((groups + 2) * 2.0 ** -22 * sizes).amax(1)                               # of any logit of the token
    off_loss = 2 * off + 2.0 ** -20 * (1 + losses.abs())                            # exponentials and logarithm of 2^-22 each
    if reduction == "none":
        _check("loss", loss.detach().flatten(), losses, off_loss)
    else:
        total = losses.sum() / (counts if reduction == "mean" else 1)
        _check("loss", loss.detach(), total, off_loss.sum() / (counts if reduction == "mean" else 1))
    ok = _half_step(product) if product != F32 else 2.0 ** -22                      # the rounding of dz
    g_max = float(g.abs().max())
    lost = (2.0 ** -39 if product == F16 else 2.0 ** -126) * g_max                  # fp16: half the smallest step, over 2^14; exponentials below 2^-126 are 0
    # beside what is relative to dz: at the target, p - 1 of a p near 1 has the whole error of p, which is an exponential of 2^-22 (the
    # instruction's bound is 2^-22.5) over a sum of such exponentials: 2^-21
    counts = targets.flatten() != ignore
    at_target = torch.zeros_like(dz).scatter_(1, torch.where(counts, targets.flatten(), 0)[:, None], 2.0 ** -21)
    each = dz.abs() * (ok + 2 * off[:, None] + 2.0 ** -20) + (g.abs() * counts)[:, None] * at_target + lost

    def around(a, abs_a, e, b, k):
        many = (-(-k // 64) * 4 + 70) if product != F32 else 32 * 4 + 200           # groups in one sum; fp32 leaves tensor memory every 2,048
        return a @ b, e @ b.abs() + many * 2.0 ** -22 * (abs_a @ b.abs())

    want, slack = around(dz, dz.abs(), each, rw.detach().double(), vocab)
    _check("dx", dx.reshape(-1, width), want, slack)
    if train:                                               # x over the sum of exponentials is rounded too
        each = each + dz.abs() * ok
    want, slack = around(dz.T, dz.T.abs(), each.T, rx.detach().double(), n)
    _check("dw", dw, want, slack)
    assert _lib.device_status() == 0
    return loss, dx, dw


LOSSES = [
    # tokens, vocab, width, reduction
    (1, 1, 1, "sum"), (1, 2, 8, "mean"), (3, 17, 5, "none"), (16, 1000, 64, "none"), (127, 129, 63, "sum"), (128, 128, 128, "mean"),
    (129, 257, 65, "none"), (200, 3001, 200, "mean"), (257, 513, 72, "none"), (300, 9000, 256, "sum"), (700, 5000, 520, "mean"),
    (2500, 700, 40, "mean"), (40, 40000, 136, "none"),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,vocab,width,reduction", LOSSES)
def test_loss_and_its_gradients(tokens, vocab, width, reduction, dtype):
    gen = _gen(tokens * 7 + vocab)
    x = _randn(gen, tokens, width, dtype=dtype)
    w = _randn(gen, vocab, width, dtype=dtype, scale=2.0 / math.sqrt(width))
    targets = torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    if tokens > 2:
        targets[1::7] = -100
    _check_loss(x, w, targets, reduction)
    if dtype != F16:
        _check_loss(x, w, targets, "mean" if reduction == "none" else reduction, train=True)


@pytest.mark.parametrize("dtype,tokens,vocab,width,reduction", [
    (BF16, 9000, 40000, 64, "none"), (F32, 5000, 12000, 72, "none"), (F16, 9000, 40000, 64, "mean"),      # pieces of the vocabulary
    (BF16, 9000, 40000, 64, "mean"), (F32, 5000, 12000, 72, "sum"), (BF16, 1500, 262144, 16, "mean")])    # runs of tokens
def test_loss_in_several_parts(dtype, tokens, vocab, width, reduction):
    """More logits than the workspace holds at a time: 320 to 480 MB in 16 bits."""
    gen = _gen(11)
    x = torch.randn(tokens, width, device="cuda").to(dtype)
    w = (torch.randn(vocab, width, device="cuda") * 0.3).to(dtype)
    targets = torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    targets[5::11] = -100
    _check_loss(x, w, targets, reduction)
    if reduction != "none" and dtype != F16:
        _check_loss(x, w, targets, reduction, train=True)


@pytest.mark.parametrize("dtype,width,reduction", [
    (BF16, 259, "none"), (F16, 262, "sum"), (BF16, 261, "mean"), (BF16, 264, "none"), (F32, 65, "mean")])
def test_rows_of_gradients_that_start_anywhere(dtype, width, reduction):
    """Tiles enough that most are stored whole, in several pieces or runs, into rows that start at 2, 4, 8 or 16 bytes."""
    gen = _gen(12)
    tokens, vocab = (19500, 19201) if dtype != F32 else (5000, 19201)
    x = torch.randn(tokens, width, device="cuda").to(dtype)
    w = (torch.randn(vocab, width, device="cuda") * 0.2).to(dtype)
    targets = torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    targets[5::11] = -100
    _check_loss(x, w, targets, reduction)
    if dtype != F16:
        _check_loss(x, w, targets, "sum", train=True)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_of_more_tokens_than_a_run(reduction):
    """65,536 tokens' half tiles are kept at a time."""
    gen = _gen(33)
    x, w = torch.randn(70001, 24, device="cuda").bfloat16(), (torch.randn(300, 24, device="cuda") * 0.4).bfloat16()
    targets = torch.randint(0, 300, (70001,), generator=gen).cuda()
    targets[65000:66000] = -100
    _check_loss(x, w, targets, reduction)
    with torch.no_grad():
        got = layers.linear_cross_entropy(x, w, targets, reduction=reduction)
    want = torch.nn.functional.cross_entropy((x.double() @ w.double().T), targets, reduction=reduction)
    assert (got.double() - want).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_targets_that_are_all_but_impossible(dtype):
    """Losses beyond 44, where exponentials over the target's leave their range: the rows go through the product once more."""
    gen = _gen(31)
    x, w = _randn(gen, 300, 72, dtype=dtype), _randn(gen, 900, 72, dtype=dtype, scale=4.0)
    targets = torch.randint(0, 900, (300,), generator=gen).cuda()
    targets[::9] = -100
    z = x.double() @ w.double().T
    targets[1::9] = z[1::9].argmin(1)                       # up to 200
    targets[2::9] = z[2::9].argmax(1)
    losses = layers.linear_cross_entropy(x, w, targets, reduction="none")
    assert float(losses.max()) > 100 and int((losses > 44).sum()) > 30 and int((losses < 1).sum()) > 30
    for reduction, train in (("sum", True), ("sum", False), ("none", False)):
        _check_loss(x, w, targets, reduction, train=train)
    far = torch.full_like(targets[:1], int(z[1].argmin()))
    for train in (False, True):
        _check_loss(x[1:2], w, far, "mean", train=train)


def test_loss_of_batches_strides_and_padding():
    gen = _gen(12)
    base = _randn(gen, 4, 60, 2 * 128, dtype=BF16)
    table = _randn(gen, 500, 160, dtype=BF16, scale=0.2)
    targets = torch.randint(0, 500, (4, 60), generator=gen).cuda()
    targets[2] = -7                                         # a sequence of padding
    targets[0, 50:] = -7
    for x, w in ((base[..., 128:], table[:, 16:144]), (base[..., 1:129], table[:, 3:131]), (base[..., ::2], table[:, 16:144].t().contiguous().t())):
        for train in (False, True):
            if train and (x.stride(-1) != 1 or w.stride(-1) != 1):
                continue                                    # the C entries take rows
            loss, dx, dw = _check_loss(x, w, targets, "mean", ignore=-7, train=train)
            assert (dx[2] == 0).all() and (dx[0, 50:] == 0).all()
    same = _check_loss(base[:1, :1, 128:].expand(4, 60, 128), table[:, 16:144], targets, "none", ignore=-7)[0]
    assert (same[2] == 0).all()


@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_cotangents_rounding_moves_no_gradient(dtype, reduction):
    """Targets' gradients of the logits about half a step from a number of the type: rounded, they would move every token's alike, by 0.7
    to 1 half steps."""
    dloss = (1 + _half_step(dtype)) / (1 - 1 / 700) * (200 if reduction == "mean" else 1)
    gen = _gen(41)
    x, w = _randn(gen, 200, 136, dtype=dtype).requires_grad_(True), _randn(gen, 700, 136, dtype=dtype, scale=0.05).requires_grad_(True)
    targets = torch.randint(0, 700, (200,), generator=gen).cuda()
    loss = layers.linear_cross_entropy(x, w, targets, reduction=reduction)
    g = torch.full_like(loss, dloss).detach()
    (dx,) = torch.autograd.grad(loss, x, g)
    with torch.no_grad():
        z = x.double() @ w.double().T
        dz = (torch.softmax(z, 1) - torch.nn.functional.one_hot(targets, 700)) * (dloss / (200 if reduction == "mean" else 1))
        want = dz @ w.double()
    # 27,200 roundings of dx, spread over half a step or less each way: 3^-1/2 of one in their norm at most; of dz, those of what is not at
    # the target, a 15th of dx's norm
    assert float((dx.double() - want).norm() / want.norm()) < (3 ** -0.5 + 0.07) * _half_step(dtype)


@pytest.mark.parametrize("tokens,reduction", [(1, "sum"), (9, "mean"), (64, "none"), (65, "none"), (128, "sum")])
def test_few_tokens_gradients_are_as_exact_as_their_type(tokens, reduction):
    gen = _gen(42)
    x, w = _randn(gen, tokens, 272, dtype=BF16).requires_grad_(True), _randn(gen, 300, 272, dtype=BF16, scale=0.2).requires_grad_(True)
    targets = torch.randint(0, 300, (tokens,), generator=gen).cuda()
    loss = layers.linear_cross_entropy(x, w, targets, reduction=reduction)
    g = (torch.rand(loss.shape, generator=gen) + 0.5).cuda()
    (dw,) = torch.autograd.grad(loss, w, g)
    z = x.detach().double() @ w.detach().double().T
    dz = torch.softmax(z, 1) - torch.nn.functional.one_hot(targets, 300)
    want = (dz * (g if reduction == "none" else g / (tokens if reduction == "mean" else 1)).double().reshape(-1, 1)).T @ x.detach().double()
    # dz keeps 16 bits; the 81,600 roundings of dw are spread as above
    assert float((dw.double() - want).norm() / want.norm()) < (3 ** -0.5 + 0.01) * _half_step(BF16)


def test_what_is_ignored_may_be_anything():
    gen = _gen(13)
    x = _randn(gen, 90, 96, dtype=BF16)
    w = _randn(gen, 300, 96, dtype=BF16, scale=0.2)
    targets = torch.randint(0, 300, (90,), generator=gen).cuda()
    targets[::3] = 5                                        # an index of the vocabulary that counts for nothing
    clean = _check_loss(x, w, targets, "mean", ignore=5)
    clean_c = _check_loss(x, w, targets, "mean", ignore=5, train=True)
    x[::3] = float("nan")
    x[3], x[6] = float("inf"), -float("inf")
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = layers.linear_cross_entropy(a, b, targets, ignore_index=5)
    dloss = torch.tensor(0.75, device="cuda")
    dx, dw = torch.autograd.grad(loss, (a, b), dloss)
    assert torch.equal(loss, clean[0]) and torch.equal(dx, clean[1]) and torch.equal(dw, clean[2])
    assert all(torch.equal(p, q) for p, q in zip(_with_the_loss(x, w, targets, 5, "mean", BF16, dloss), clean_c))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_no_token_counts(dtype):
    x = torch.randn(20, 64, device="cuda", dtype=dtype, requires_grad=True)
    w = torch.randn(50, 64, device="cuda", dtype=dtype, requires_grad=True)
    targets = torch.full((20,), -100, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = layers.linear_cross_entropy(x, w, targets, reduction=reduction)
        assert torch.isnan(loss).all() if reduction == "mean" else (loss == 0).all()
        for grad in torch.autograd.grad(loss.sum(), (x, w)):
            assert (grad == 0).all()
        if reduction != "none" and dtype != F16:
            loss, dx, dw = _with_the_loss(x, w, targets, -100, reduction, dtype, torch.ones((), device="cuda"))
            assert (torch.isnan(loss) if reduction == "mean" else loss == 0) and (dx == 0).all() and (dw == 0).all()
    empty = layers.linear_cross_entropy(x[:0], w, targets[:0], reduction="none")
    assert empty.shape == (0,)
    assert float(layers.linear_cross_entropy(x[:0], w, targets[:0], reduction="sum").detach()) == 0.0
    assert torch.isnan(layers.linear_cross_entropy(x[:0], w, targets[:0]))
    (dw,) = torch.autograd.grad(layers.linear_cross_entropy(x[:0], w, targets[:0], reduction="sum"), (w,))
    assert dw.shape == w.shape and (dw == 0).all()


def test_targets_outside_the_vocabulary_and_values_that_are_not_finite():
    gen = _gen(14)
    x, w = _randn(gen, 10, 64, dtype=BF16), _randn(gen, 30, 64, dtype=BF16)
    targets = torch.randint(0, 30, (10,), generator=gen).cuda()
    want = layers.linear_cross_entropy(x, w, targets, reduction="none")
    targets[3], targets[4], targets[5] = 30, -1, 1 << 40
    a = x.clone().requires_grad_(True)
    got = layers.linear_cross_entropy(a, w, targets, reduction="none")
    bad = torch.zeros(10, dtype=torch.bool, device="cuda")
    bad[3:6] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad].detach(), want[~bad])
    (dx,) = torch.autograd.grad(got, (a,), torch.ones_like(got))
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    loss, dx, dw = _with_the_loss(x, w, targets, -100, "sum", BF16, torch.ones((), device="cuda"))
    assert torch.isnan(loss) and torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all() and torch.isnan(dw).all()
    targets = torch.randint(0, 30, (10,), generator=gen).cuda()
    a = x.clone()
    a[2, 5], a[7, 1] = float("nan"), float("inf")
    got = layers.linear_cross_entropy(a, w, targets, reduction="none")
    assert torch.isnan(got[2]) and not torch.isfinite(got[7]) and torch.isfinite(got[[0, 1, 3, 4, 5, 6, 8, 9]]).all()


def test_masked_words():
    """Rows of the table that push their logits to the end of the type, or to -inf in the sum, leave the others alone."""
    gen = _gen(15)
    x = _randn(gen, 150, 64, dtype=BF16).abs() + 0.1
    w = _randn(gen, 700, 64, dtype=BF16, scale=0.2)
    targets = torch.randint(0, 300, (150,), generator=gen).cuda()
    w[300:] = torch.finfo(BF16).min                         # sums overflow to -inf: words that are never said
    got = layers.linear_cross_entropy(x, w, targets, reduction="none")
    want = layers.linear_cross_entropy(x, w[:300], targets, reduction="none")
    assert torch.isfinite(got).all() and (got - want).abs().max() < 2.0 ** -18
    w[:] = torch.finfo(BF16).min                            # whole tiles of nothing but -inf, in front and behind
    w[650] = 0.01
    got = layers.linear_cross_entropy(x, w, torch.full_like(targets, 650), reduction="none")
    assert (got.abs() < 2.0 ** -18).all()


def test_small_and_large_cotangents_in_fp16():
    """Cotangents of a loss scale, and tokens whose weights lie 2^15 apart: dz keeps its bits."""
    gen = _gen(16)
    x, w = _randn(gen, 60, 64, dtype=F16), _randn(gen, 200, 64, dtype=F16, scale=0.2)
    targets = torch.randint(0, 200, (60,), generator=gen).cuda()
    a = x.clone().requires_grad_(True)
    loss = layers.linear_cross_entropy(a, w, targets, reduction="none")
    g = torch.ones(60, device="cuda") * 65536.0
    g[::2] = 2.0
    (dx,) = torch.autograd.grad(loss, (a,), g)
    _, dz, _ = _loss_reference(x, w, targets, -100, g.double())
    want = dz @ w.double()
    inside = want.abs() < 65504
    assert float(((dx.double() - want) * inside).abs().sum(1).div((want * inside).abs().sum(1)).max()) < 2.0 ** -9


def test_gradients_agree_with_differences():
    gen = _gen(17)
    x, w = _randn(gen, 30, 40).requires_grad_(True), _randn(gen, 90, 40, scale=0.3).requires_grad_(True)
    targets = torch.randint(0, 90, (30,), generator=gen).cuda()
    dx, dw = torch.autograd.grad(layers.linear_cross_entropy(x, w, targets, reduction="sum"), (x, w))
    h = 2.0 ** -6
    for leaf, grad in ((0, dx), (1, dw)):
        u = torch.sign(grad)
        at = lambda s: layers.linear_cross_entropy(x + s * u, w, targets, reduction="sum") if leaf == 0 else \
            layers.linear_cross_entropy(x, w + s * u, targets, reduction="sum")  # noqa: E731
        with torch.no_grad():
            slope = float((8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))).double() / (12 * h))
        want = float((grad.double() * u).sum())
        assert abs(slope - want) < 2e-3 * abs(want)         # the fourth difference's error, h^4, and 2^-22 of a sum of ~150 over h


@pytest.mark.parametrize("product", [BF16, F16])
def test_autocast_rounds_the_operands_and_keeps_the_gradients_types(product):
    gen = _gen(18)
    x, w = _randn(gen, 300, 136, dtype=BF16), _randn(gen, 1100, 136, scale=0.2)
    targets = torch.randint(0, 1100, (300,), generator=gen).cuda()
    with torch.autocast("cuda", dtype=product):
        _check_loss(x, w, targets, "mean", product=product)
        _check_loss(x.float(), w.bfloat16(), targets, "sum", product=product)
    if product == BF16:
        _check_loss(x, w, targets, "mean", product=product, train=True)
        _check_loss(x.float(), w.bfloat16(), targets, "sum", product=product, train=True)


def test_only_one_gradient_is_asked_for():
    gen = _gen(19)
    x, w = _randn(gen, 200, 72, dtype=BF16).requires_grad_(True), _randn(gen, 900, 72, dtype=BF16).requires_grad_(True)
    targets = torch.randint(0, 900, (200,), generator=gen).cuda()
    both = torch.autograd.grad(layers.linear_cross_entropy(x, w, targets), (x, w))
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x, w.detach(), targets), (x,))[0], both[0])
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x.detach(), w, targets), (w,))[0], both[1])
    loss = layers.linear_cross_entropy(x, w, targets)
    assert torch.equal(torch.autograd.grad(loss, (x,), retain_graph=True)[0], both[0]) and torch.equal(torch.autograd.grad(loss, (w,))[0], both[1])


def test_large_problems_of_one_cotangent():
    """Large enough that the Python call computes the gradients with the loss: one gradient or both, one cotangent or another, twice, an
    empty rest of a batch, a captured step, other memory beneath the saved sums."""
    gen = _gen(32)
    x = torch.randn(6100, 256, device="cuda").bfloat16().requires_grad_(True)
    w = (torch.randn(50000, 256, device="cuda") * 0.2).bfloat16().requires_grad_(True)
    targets = torch.randint(0, 50000, (6100,), generator=gen).cuda()
    assert _prefers(x, w, targets, -100, "mean", BF16)
    loss = layers.linear_cross_entropy(x, w, targets)
    both = torch.autograd.grad(loss, (x, w), retain_graph=True)
    _check_loss(x, w, targets, "mean")
    assert all(torch.equal(2 * a, b) for a, b in zip(both, torch.autograd.grad(loss, (x, w), torch.tensor(2.0, device="cuda"))))
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x, w.detach(), targets), (x,))[0], both[0])
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x.detach(), w, targets), (w,))[0], both[1])
    with torch.no_grad():
        assert abs(float(layers.linear_cross_entropy(x, w, targets)) - float(loss.detach())) < 1e-5
    with torch.autograd.graph.save_on_cpu():
        loss = layers.linear_cross_entropy(x, w, targets)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), both))
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, odd):
        loss = layers.linear_cross_entropy(x, w, targets)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w)), both))
    (g,) = torch.autograd.grad(layers.linear_cross_entropy(x, w, targets), x, torch.ones((), device="cuda", requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layers.linear_cross_entropy(x, w, targets), (x, w))
    torch.cuda.current_stream().wait_stream(side)
    del loss, g
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(layers.linear_cross_entropy(x, w, targets), (x, w))
    targets[100:400] = -100
    graph.replay()
    want = torch.autograd.grad(layers.linear_cross_entropy(x, w, targets), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(captured, want)) and (want[0][100:400] == 0).all()
    assert _lib.device_status() == 0


# ---- as the rest of torch uses them ------------------------------------------------------------------------------------------------

def _step(idx, table, weight, targets):
    """Embedding, norms and the loss on the same table."""
    x = layers.embedding(idx, table, scale=2.0)
    s, y = layers.add_layer_norm(x, x.square(), weight)
    return layers.linear_cross_entropy(layers.layer_norm(s + y, weight), table, targets)


def _step_inputs(seed, dtype=BF16):
    gen = _gen(seed)
    return (torch.randint(0, 400, (2, 70), generator=gen).cuda(), _randn(gen, 400, 136, dtype=dtype, scale=0.5),
            _randn(gen, 136, dtype=dtype, mean=1.0, scale=0.1), torch.randint(0, 400, (2, 70), generator=gen).cuda())


def test_together_they_agree_with_the_library_operators():
    idx, table, weight, targets = _step_inputs(20, F32)
    leaves = [table.requires_grad_(True), weight.requires_grad_(True)]
    got = _step(idx, table, weight, targets)
    grads, got = torch.autograd.grad(got, leaves), got.detach()
    t64, w64 = (t.detach().double().requires_grad_(True) for t in leaves)
    x = t64[idx] * 2.0
    s = x + x.square()
    y = torch.nn.functional.layer_norm(s, (136,), w64)
    h = torch.nn.functional.layer_norm(s + y, (136,), w64)
    want = torch.nn.functional.cross_entropy((h @ t64.T).reshape(-1, 400), targets.reshape(-1))
    wanted = torch.autograd.grad(want, (t64, w64))
    assert abs(float(got) - float(want.detach())) < 1e-5 * float(want.detach())
    for a, b in zip(grads, wanted):
        assert float((a.double() - b).norm() / b.norm()) < 1e-5


def test_calls_are_the_same_from_time_to_time_and_on_other_streams():
    first, second = _step_inputs(21), _step_inputs(22)
    want = []
    for idx, table, weight, targets in (first, second):
        leaves = [table.requires_grad_(True), weight.requires_grad_(True)]
        loss = _step(idx, table, weight, targets)
        want.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (inputs, stream) in enumerate(zip((first, second), streams)):
            with torch.cuda.stream(stream):
                loss = _step(*inputs)
                got[i] = [loss.detach(), *torch.autograd.grad(loss, inputs[1:3])]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_captured_step_follows_its_inputs():
    idx, table, weight, targets = _step_inputs(23)
    table.requires_grad_(True)
    weight.requires_grad_(True)
    # no eager graph of the leaves may live while a backward is captured: torch would sum their gradients on its stream
    eager = float(_step(idx, table, weight, targets).detach())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_step(idx, table, weight, targets), (table, weight))
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        loss = _step(idx, table, weight, targets)
        grads = torch.autograd.grad(loss, (table, weight))
    for seed in (24, 25):
        new = _step_inputs(seed)
        with torch.no_grad():
            for to, source in zip((idx, table, weight, targets), new):
                to.copy_(source)
        graph.replay()
        want = _step(idx, table, weight, targets)
        for a, b in zip((loss, *grads), (want, *torch.autograd.grad(want, (table, weight)))):
            assert torch.equal(a, b)
    assert math.isfinite(eager)


def test_saved_tensors_may_be_moved_and_hooks_see_them():
    idx, table, weight, targets = _step_inputs(26)
    leaves = [table.requires_grad_(True), weight.requires_grad_(True)]
    want = torch.autograd.grad(_step(idx, table, weight, targets), leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = _step(idx, table, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), want))
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, odd):
        loss = _step(idx, table, weight, targets)
    for a, b in zip(torch.autograd.grad(loss, leaves), want):
        assert (a.float() - b.float()).norm() < 2.0 ** -7 * b.float().norm()        # other loads, another order


def test_a_tensor_that_was_changed_since_is_noticed_and_a_second_derivative_is_refused():
    idx, table, weight, targets = _step_inputs(27)
    table.requires_grad_(True)
    loss = layers.linear_cross_entropy(layers.embedding(idx, table), table, targets, reduction="none").sum()
    with torch.no_grad():
        table.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    for out in (layers.layer_norm(x).square().sum(), layers.linear_cross_entropy(x, torch.randn(9, 32, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")),
                layers.embedding(targets[0, :3] % 4, x).square().sum()):
        (g,) = torch.autograd.grad(out, x, create_graph=True)
        if g.requires_grad:
            with pytest.raises(RuntimeError, match="once_differentiable"):
                g.sum().backward()


@pytest.mark.filterwarnings("ignore")
def test_traces_and_transforms_are_refused():
    x, w = torch.randn(4, 32, device="cuda"), torch.randn(9, 32, device="cuda")
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    for call, arg in ((layers.layer_norm, x), (lambda a: layers.linear_cross_entropy(a, w, t), x), (lambda a: layers.embedding(t, a), w)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (arg,), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda a: call(a).sum())(arg)


def test_refusals_name_what_is_wrong():
    x, w = torch.randn(4, 32, device="cuda"), torch.randn(9, 32, device="cuda")
    t = torch.zeros(4, dtype=torch.long, device="cuda")
    for match, call in (
            ("CUDA", lambda: layers.layer_norm(x, w[0].cpu())), ("dtype", lambda: layers.layer_norm(x.double())),
            ("dtype", lambda: layers.layer_norm(x, dtype=torch.int32)), ("must be \\(32", lambda: layers.layer_norm(x, w[0, :31])),
            ("one dtype", lambda: layers.layer_norm(x, w[0], w[0].half())), ("eps", lambda: layers.layer_norm(x, eps=-1.0)),
            ("16384", lambda: layers.layer_norm(torch.zeros(2, 16385, device="cuda"))), ("one shape", lambda: layers.add_layer_norm(x, x[:3])),
            ("int64", lambda: layers.embedding(t.float(), w)), ("vocab, width", lambda: layers.embedding(t, w[0])), ("CUDA", lambda: layers.embedding(t.cpu(), w)),
            ("dtype", lambda: layers.embedding(t, w.double())), ("width", lambda: layers.linear_cross_entropy(x, w[:, :31], t)),
            ("shape", lambda: layers.linear_cross_entropy(x, w, t[:3])), ("dtype", lambda: layers.linear_cross_entropy(x.half(), w, t)),
            ("int64", lambda: layers.linear_cross_entropy(x, w, t.float())), ("reduction", lambda: layers.linear_cross_entropy(x, w, t, reduction="max")),
            ("CUDA", lambda: layers.linear_cross_entropy(x, w.cpu(), t))):
        with pytest.raises(ValueError, match=match):
            call()
