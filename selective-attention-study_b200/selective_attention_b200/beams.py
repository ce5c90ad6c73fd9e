"""Beam search over a decoder with Selective Attention: the selection of the best continuations.

The states follow with ``paged.reorder_rows`` and ``paged.move_rows``: a beam's history sums belong to its own queries, so beams
share pages of keys and values but never a history."""

from __future__ import annotations

import torch

from . import _lib


def beam_select(logits: torch.Tensor, scores: torch.Tensor, width: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``width`` (at most 32) best continuations of every group of beams: ``scores[g, k] + log_softmax(logits[g, k])[v]``, largest
    first, equal ones by the lowest (k, v).

    logits: (groups, beams, vocab) fp32, bf16 or fp16, any group and beam strides; scores: (groups, beams), finite, or -inf for
    a beam that does not take part.  Returns the new scores (groups, width) fp32, the row that each comes from (int32, counted
    over all groups: ``parents`` of ``paged.reorder_rows`` where every group has ``width`` rows), and its token (int64).
    Compared in 64 bits, over log-sum-exps of 32-bit exponentials (2^-20 at most): continuations of two beams that are nearer to one
    another than that may come in either order, and so may those of one beam that 64 bits do not tell apart (a score of -1e30, say).
    Where a beam's logits hold a NaN or +inf, or nothing above -inf, its continuations count as -inf."""
    return _lib.native().beam_select(logits, scores, int(width))
