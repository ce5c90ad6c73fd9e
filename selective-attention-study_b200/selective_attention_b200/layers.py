"""What a decoder with Selective Attention has around its attention: layer norm, the embedding, and the loss over the vocabulary.

The reference calls library operators here (``src/selective_attention/model.py:31-47,325-328,365-366,402-418``); its loss keeps the
(tokens, vocab) logits, in pieces for evaluation (``:420-447``).  Here they are kernels of the library, differentiable once, with gradients
that are the same from call to call.  CUDA tensors and the built library only; float32, bfloat16 and float16, any strides (a tensor whose
last axis is not contiguous is copied).  A call cannot be recorded by ``torch.jit.trace`` and has no forward-mode derivative: a tensor that
carries a tangent is refused."""

from __future__ import annotations

import torch

from . import _lib

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               dtype: torch.dtype | None = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis, of 1 to 16,384 values, with statistics in 32 bits.

    ``dtype``: of the result; by default x's (autocast does not change it).  weight and bias, either may be None, have one dtype,
    which need not be x's; their gradients have it too."""
    return _lib.native().layer_norm(x, None, weight, bias, float(eps), dtype)[0]


def add_layer_norm(x: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   eps: float = 1e-5, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(x + branch, its ``layer_norm``): the residual sum and the norm behind it, in one pass in either direction.

    The sum has x's dtype; what is normalised is the sum as it is kept.  branch has x's shape and a dtype of its own, which its
    gradient has too."""
    summed, y = _lib.native().layer_norm(x, branch, weight, bias, float(eps), dtype)
    return summed, y


def embedding(idx: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[idx]`` for idx (...) int64 or int32 and weight (vocab, width): (..., width) in ``dtype``, by default weight's.

    The gradient of a row of the table sums its tokens in fp32, in their order.  An index outside the table gives a row of NaN
    and has no part in the gradient."""
    return _lib.native().embedding(idx, weight, float(scale), dtype)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``cross_entropy(x @ weight.T, targets)`` in fp32 without the logits, for x (..., width), weight (vocab, width) and targets (...)
    int64 or int32: one number, or with ``reduction="none"`` a loss for every target (0 where it is ignored).

    The forward keeps a log-sum-exp for every token; the backward computes the logits again, a piece of the vocabulary at a time.  Where
    ``reduction`` leaves one cotangent and the problem is large (bf16 and fp32 products), the gradients are computed with the loss
    instead, up to the cotangent, a product less: their sums, of x's and weight's shapes in fp32, are kept for the backward, which scales
    them.  Either way up to half a GB of what stands for logits is there at a time: more tokens go in runs, with a sum of the table's gradient in
    fp32 beside them.

    x and weight have one dtype, or under autocast are rounded to its; their gradients have their own.  bf16 and fp16 products are
    exact with fp32 sums (tensor cores round towards zero: at most 1,024 products of a logit and 8,192 of a gradient are added that way), and
    the gradient of the logits is rounded to that dtype between its products, but for the target's in x's gradient (fp16: scaled by the
    largest cotangent, so tokens whose cotangent is 2^-19 of it or less lose bits).  weight's gradient shows that rounding beside its own
    beyond 128 tokens: 2.4e-3 of its norm where bf16 by itself is 1.7e-3, 1.8e-3 where the gradients come with the loss.  fp32 operands
    are split into three bf16 parts, which keep 24 bits.

    What stands in x where a target is ignored does not matter.  A target outside the vocabulary that is not ``ignore_index`` makes its
    loss and the gradients NaN.  The mean over no target at all is NaN, its gradients are zeros."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(REDUCTIONS)}; got {reduction!r}")
    return _lib.native().linear_cross_entropy(x, weight, targets, int(ignore_index), REDUCTIONS[reduction])
