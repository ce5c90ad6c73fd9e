"""What a decoder with Selective Attention has around its attention, as cases that can be timed and compared.

Three operators of ``layers``, in a training step and, without gradients, in an answer:

    norm    ``layers.layer_norm`` and, after a residual sum, ``layers.add_layer_norm``
    embed   ``layers.embedding``: rows of the table, scaled; the gradient sums the tokens of every row
    loss    ``layers.linear_cross_entropy``: the output projection and the cross entropy over the vocabulary, whose logits are
            never kept

``run`` has each in its plain form, or (``own``) by the framework's calls.
"""

import math
import os
import sys

import torch

own = False
PACKAGE = os.path.join(os.getcwd(), "selective-attention-study_b200")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _framework():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from selective_attention_b200 import layers

    return layers


# ---- cases --------------------------------------------------------------------------------------------------------------------

def _norm(name=None, *, rows, width, x, y, branch="", bias=False, train=True, eps=1e-5):
    """``x``, ``branch``, ``y``: types of the input, of what is added to it first ("": nothing) and of the result; parameters are
    fp32 beside an fp32 input and of its type otherwise."""
    c = dict(kind="norm", rows=rows, width=width, x=x, y=y, branch=branch, bias=bias, train=train, eps=eps)
    return c if name is None else dict(c, name=name)


def _embed(name=None, *, tokens, vocab, width, dtype, y, scale=1.0, train=True, skew=1.0):
    """``skew``: exponent of the tokens' frequencies by their rank (1: as words come; 0: evenly)."""
    c = dict(kind="embed", tokens=tokens, vocab=vocab, width=width, dtype=dtype, y=y, scale=scale, train=train, skew=skew)
    return c if name is None else dict(c, name=name)


def _loss(name=None, *, tokens, vocab, width, dtype, reduction="mean", ignored=0.0, train=True, spread=3.0):
    """``ignored``: share of tokens that do not count; ``spread``: standard deviation of a token's logits."""
    c = dict(kind="loss", tokens=tokens, vocab=vocab, width=width, dtype=dtype, reduction=reduction, ignored=ignored, train=train,
             spread=spread)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # a decode step of eight requests of the 12-head model: latency
        _norm("norm-8-rows", rows=8, width=768, x="bf16", y="bf16", train=False),
        # the residual sum and the norm after it, in training at 16K context: an fp32 residual stream and bf16 branches
        _norm("add-norm-16k", rows=16384, width=1024, x="fp32", y="bf16", branch="bf16"),
        # fp16 activations of an odd width, with a bias
        _norm("norm-odd-fp16", rows=3001, width=1027, x="fp16", y="fp16", bias=True),
        # a batch of narrow rows
        _norm("norm-narrow", rows=50000, width=200, x="bf16", y="bf16"),
        # a prompt's tokens out of a bf16 table, scaled by the root of the width
        _embed("embed-prompt-300", tokens=300, vocab=50304, width=768, dtype="bf16", y="bf16", scale=math.sqrt(768.0), train=False),
        # the table of the 16-head model in training at 16K context, words as often as words are
        _embed("embed-16k", tokens=16384, vocab=50304, width=1024, dtype="fp32", y="fp32"),
        # a small table that every token of a long batch falls into: the longest sums
        _embed("embed-bytes", tokens=40000, vocab=257, width=520, dtype="bf16", y="bf16"),
        # how likely 16 candidate tokens are, one of each request
        _loss("score-16", tokens=16, vocab=50304, width=1024, dtype="bf16", reduction="none", train=False),
        # the loss of a 2K batch of the 12-head model, a tenth of it padding
        _loss("loss-2k", tokens=2048, vocab=50304, width=768, dtype="bf16", ignored=0.1),
        # the loss of the decoder's training step at 16K context
        _loss("loss-16k", tokens=16384, vocab=50304, width=1024, dtype="bf16"),
        # a small fp32 model
        _loss("loss-fp32", tokens=1000, vocab=8003, width=520, dtype="fp32", reduction="sum", ignored=0.05),
        # fp16, every token with a weight of its own
        _loss("loss-weighted-fp16", tokens=777, vocab=32001, width=1000, dtype="fp16", reduction="none"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "embed", "embed", "loss", "loss", "loss"])
    train = rng.random() < 0.7
    if kind == "norm":
        width = _log(rng, 3, 9000)
        x = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        half = rng.choice(["bf16", "fp16"]) if x == "fp32" else x
        return _norm(rows=_log(rng, 1, max(1, 16_000_000 // width)), width=width, x=x, y=rng.choice([x, half]),
                     branch=rng.choice(["", x, half]), bias=rng.random() < 0.3, train=train, eps=rng.choice([1e-5, 1e-6]))
    if kind == "embed":
        width, dtype = _log(rng, 1, 4096), rng.choice(["fp32", "bf16", "fp16"])
        return _embed(tokens=_log(rng, 1, min(60000, 16_000_000 // width)), vocab=_log(rng, 1, min(100_000, 50_000_000 // width)),
                      width=width, dtype=dtype, y=rng.choice([dtype, dtype, "bf16"]) if dtype == "fp32" else dtype,
                      scale=rng.choice([1.0, 1.0, math.sqrt(width)]), train=train, skew=rng.choice([1.0, 1.0, 0.0, 2.0]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    width = _log(rng, 8, 1024 if dtype == "fp32" else 4096)
    vocab = _log(rng, 3, 30_000 if dtype == "fp32" else 130_000)
    most = (10**11 if dtype == "fp32" else 7 * 10**11) // (width * vocab)
    return _loss(tokens=_log(rng, 1, max(1, min(most, 16384 if dtype != "fp32" else 4096))), vocab=vocab, width=width, dtype=dtype,
                 reduction=rng.choice(["mean", "mean", "sum", "none"]), ignored=rng.choice([0.0, 0.0, 0.1, 0.5]), train=train,
                 spread=rng.choice([0.6, 3.0]))


# ---- the state that a program has in hand ------------------------------------------------------------------------------------

def _normal(gen, shape, scale=1.0, dtype="fp32", mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + mean).to(DTYPES[dtype])


def prepare(case, seed):
    c, gen = case, torch.Generator("cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "norm":
        n, d = c["rows"], c["width"]
        kind = "fp32" if c["x"] == "fp32" else c["x"]
        s["x"] = _normal(gen, (n, d), 2.0, c["x"], mean=0.3)
        s["branch"] = _normal(gen, (n, d), 0.5, c["branch"]) if c["branch"] else None
        s["weight"] = _normal(gen, (d,), 0.2, kind, mean=1.0)
        s["bias"] = _normal(gen, (d,), 0.2, kind) if c["bias"] else None
        if c["train"]:
            s["dy"] = _normal(gen, (n, d), 1.0, c["y"])
            s["dsum"] = _normal(gen, (n, d), 1.0, c["x"]) if c["branch"] else None
    elif c["kind"] == "embed":
        n, v, d = c["tokens"], c["vocab"], c["width"]
        rank = torch.arange(1, v + 1, device="cuda", dtype=torch.float64)
        upto = torch.cumsum(rank ** -c["skew"], 0)
        at = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * upto[-1]
        word = torch.randperm(v, generator=gen, device="cuda")                  # frequent words stand anywhere in the table
        s["idx"] = word[torch.searchsorted(upto, at).clamp_(max=v - 1)]
        s["weight"] = _normal(gen, (v, d), 0.02, c["dtype"])
        if c["train"]:
            s["dy"] = _normal(gen, (n, d), 1.0, c["y"])
    else:
        n, v, d = c["tokens"], c["vocab"], c["width"]
        s["x"] = _normal(gen, (n, d), 1.0, c["dtype"])
        s["weight"] = _normal(gen, (v, d), c["spread"] / math.sqrt(d), c["dtype"])
        targets = torch.randint(0, v, (n,), generator=gen, device="cuda")
        s["targets"] = torch.where(torch.rand(n, generator=gen, device="cuda") < c["ignored"], -100, targets)
        if c["reduction"] == "mean" and n:
            s["targets"][0] = targets[0]                                        # a batch has a token that counts
        if c["train"]:
            g = torch.rand(n, generator=gen, device="cuda") + 0.5
            s["dloss"] = g if c["reduction"] == "none" else g[0] * (1024.0 if c["dtype"] == "fp16" else 1.0)
    if c["train"]:
        for name in ("x", "branch", "weight", "bias"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(state):
    return {"norm": _run_norm, "embed": _run_embed, "loss": _run_loss}[state["case"]["kind"]](state)


def _run_norm(s):
    c = s["case"]
    dtype = DTYPES[c["y"]]
    if own:
        layers = _framework()
        if s["branch"] is None:
            out = [layers.layer_norm(s["x"], s["weight"], s["bias"], eps=c["eps"], dtype=dtype)]
        else:
            out = list(layers.add_layer_norm(s["x"], s["branch"], s["weight"], s["bias"], eps=c["eps"], dtype=dtype))
        if not c["train"]:
            return out
        leaves = [t for t in (s["x"], s["branch"], s["weight"], s["bias"]) if t is not None]
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, ([] if s["branch"] is None else [s["dsum"]]) + [s["dy"]]))
    x = s["x"].detach().float()
    if s["branch"] is not None:
        summed = (x + s["branch"].detach().float()).to(s["x"].dtype)
        x = summed.float()
    w = s["weight"].detach().float()
    off = x - x.mean(1, keepdim=True)
    r = (off.square().mean(1, keepdim=True) + c["eps"]).rsqrt()
    h = off * r
    y = h * w if s["bias"] is None else h * w + s["bias"].detach().float()
    out = ([] if s["branch"] is None else [summed]) + [y.to(dtype)]
    if not c["train"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    if s["branch"] is not None:
        dx = dx + s["dsum"].float()
    out.append(dx.to(s["x"].dtype))
    if s["branch"] is not None:
        out.append(dx.to(s["branch"].dtype))
    out.append((dy * h).sum(0).to(s["weight"].dtype))
    if s["bias"] is not None:
        out.append(dy.sum(0).to(s["bias"].dtype))
    return out


def _run_embed(s):
    c = s["case"]
    dtype = DTYPES[c["y"]]
    if own:
        y = _framework().embedding(s["idx"], s["weight"], scale=c["scale"], dtype=dtype)
        return [y.detach(), *torch.autograd.grad(y, s["weight"], s["dy"])] if c["train"] else [y]
    w = s["weight"].detach()
    y = (w[s["idx"]].float() * c["scale"]).to(dtype)
    if not c["train"]:
        return [y]
    dw = torch.zeros(w.shape, device="cuda").index_add_(0, s["idx"], s["dy"].float())
    return [y, (dw * c["scale"]).to(w.dtype)]


def _run_loss(s):
    c = s["case"]
    if own:
        loss = _framework().linear_cross_entropy(s["x"], s["weight"], s["targets"], reduction=c["reduction"])
        return [loss.detach(), *torch.autograd.grad(loss, (s["x"], s["weight"]), s["dloss"])] if c["train"] else [loss]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    counts = s["targets"] != -100
    at = s["targets"].clamp(min=0)[:, None]
    z = x @ w.T
    most = z.amax(1, keepdim=True)
    z = z - most
    p = z.exp()
    total = p.sum(1, keepdim=True)
    losses = torch.where(counts, total[:, 0].log() - z.gather(1, at)[:, 0], 0.0)
    del z
    share = 1.0 / counts.sum() if c["reduction"] == "mean" else 1.0
    loss = losses if c["reduction"] == "none" else losses.sum() * share
    if not c["train"]:
        return [loss]
    g = torch.where(counts, s["dloss"] * share, 0.0)[:, None]
    dz = p.mul_(g / total).scatter_add_(1, at, -g)
    return [loss, (dz @ w).to(s["x"].dtype), (dz.T @ x).to(s["weight"].dtype)]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
    c = case
    size = {"": 0, "fp32": 4, "bf16": 2, "fp16": 2}
    if c["kind"] == "norm":
        n = c["rows"] * c["width"]
        forward = size[c["x"]] * (2 if c["branch"] else 1) + size[c["branch"]] + size[c["y"]]
        backward = size[c["x"]] * (3 if c["branch"] else 2) + size[c["branch"]] + size[c["y"]]
        return {"bytes": n * (forward + (backward if c["train"] else 0)), "flops": n * (24 if c["train"] else 8)}
    if c["kind"] == "embed":
        n, table = c["tokens"] * c["width"], c["vocab"] * c["width"]
        forward = n * size[c["y"]] + min(n, table) * size[c["dtype"]] + 8 * c["tokens"]
        return {"bytes": forward + ((n * size[c["y"]] + table * size[c["dtype"]]) if c["train"] else 0), "flops": n * (2 if c["train"] else 1)}
    x, w = c["tokens"] * c["width"], c["vocab"] * c["width"]
    passes = 2 if c["train"] else 1
    return {"bytes": passes * size[c["dtype"]] * (x + w) + 12 * c["tokens"], "flops": (6 if c["train"] else 2) * c["tokens"] * w}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    s = {k: t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in s.items()}
    if c["kind"] == "norm":
        d, out = c["width"], []
        x = s["x"]
        if s["branch"] is not None:
            out.append(x + s["branch"])
            x = out[0].to(DTYPES[c["x"]]).double()                             # what is normalised is the sum as it is kept
        var, mu = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + c["eps"])
        h = (x - mu) / sd
        y = h * s["weight"]
        out.append(y if s["bias"] is None else y + s["bias"])
        if c["train"]:
            g = s["dy"] * s["weight"]
            dx = (d * g - g.sum(1, keepdim=True) - h * (g * h).sum(1, keepdim=True)) / (d * sd)
            if s["branch"] is not None:
                dx = dx + s["dsum"]
                out.append(dx)
            out += [dx, torch.einsum("nd,nd->d", s["dy"], h)]
            if s["bias"] is not None:
                out.append(s["dy"].sum(0))
        return out
    if c["kind"] == "embed":
        out = [s["weight"].index_select(0, s["idx"]) * c["scale"]]
        if c["train"]:
            order = torch.argsort(s["idx"], stable=True)
            sums = torch.cumsum(s["dy"][order], 0)
            word, count = torch.unique_consecutive(s["idx"][order], return_counts=True)
            ends = sums[torch.cumsum(count, 0) - 1]
            dw = torch.zeros_like(s["weight"])
            dw[word] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * c["scale"]
            out.append(dw)
        return out
    x, w, targets = s["x"], s["weight"], s["targets"]
    n, dx, dw, losses = c["tokens"], torch.empty_like(x), torch.zeros_like(w), []
    fine = targets.ge(0)
    share = 1.0 / float(fine.sum()) if c["reduction"] == "mean" else 1.0
    for a in range(0, n, 2048):
        b = min(n, a + 2048)
        z = torch.einsum("nd,vd->nv", x[a:b], w)
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        here, right = fine[a:b], targets[a:b].clamp(min=0)
        rows = torch.arange(b - a, device="cuda")
        losses.append(-logp[rows, right] * here)
        if c["train"]:
            g = (s["dloss"][a:b] if c["reduction"] == "none" else s["dloss"]) * share * here
            dz = logp.exp_()
            dz[rows, right] -= 1.0
            dz *= g[:, None]
            dx[a:b] = torch.einsum("nv,vd->nd", dz, w)
            dw += torch.einsum("nv,nd->vd", dz, x[a:b])
    losses = torch.cat(losses)
    loss = losses if c["reduction"] == "none" else losses.sum() * share
    return [loss, dx, dw] if c["train"] else [loss]
