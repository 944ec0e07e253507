"""Distillation of a draft model from a teacher's top log-probabilities.

The reference verifies drafts but has no way to train the drafter
(pagedmoe/mtp.py loads it from the checkpoint).  A drafter's tokens are kept
in proportion to the overlap of its distribution with the target's (verify's
residual mode); this is the loss that closes the gap, from the target's
top_logprobs alone.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L

_TAILS = {"drop": L.PM_TAIL_DROP, "bucket": L.PM_TAIL_BUCKET}
_REDUCTIONS = {"none": L.PM_REDUCE_NONE, "sum": L.PM_REDUCE_SUM, "mean": L.PM_REDUCE_MEAN}


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, temp: float = 1.0,
                 tail: str = "drop", weights: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """KL divergence of the student's distribution from a teacher's top
    log-probabilities, differentiable in the student's logits.

    logits [..., V] fp32 or bf16: the student's.  teacher_ids [..., K] int32
    or int64 and teacher_logprobs [..., K]: the teacher's most likely tokens
    and their log-probabilities at the same temperature
    (top_logprobs(teacher_logits, K, temp)); ids outside [0, V) are no
    entries, so rows may hold fewer than K.  Both are constants: no gradient
    flows into the teacher.

    With q = softmax(logits / temp):
      tail "drop":   p = the entries' probabilities divided by their sum (raw
                     logits divided by temp will do);
                     loss = sum p (log p - log q), gradient (q - p) / temp.
                     A row whose entries hold no mass has loss 0.
      tail "bucket": p as given; the teacher's remaining mass 1 - sum p is
                     matched with the student's mass outside the entries, as
                     one more outcome; that mass counts as 2**-100 at least,
                     and without a token outside the entries there is no such
                     outcome.
    The sums run over the entries as they are listed.  An id listed twice takes
    the sum of both in the gradient; in the loss they stay two outcomes of the
    teacher: it is the divergence of the sums plus p log(p / sum) of each such
    entry, a constant that may take it below 0.
    The usual factor temp ** 2 is left to the caller.

    weights [...] fp32, constants too, multiply the rows; a row of weight 0
    (padding) is not read, and neither its loss nor its gradient depends on
    what it holds.
    reduction: "mean" (divided by the sum of the weights), "sum", or "none"
    (a loss per row, [...]).

    With "mean" and "sum" the forward pass leaves the gradient behind (of the
    logits' type; the logits are not kept), so backward runs once per call.
    Capture forward and backward into one CUDA graph with torch.autograd.grad
    or leaves that no eager graph still holds.  There is no second derivative
    and no forward-mode one.  K <= 256, 4.3e-39 <= temp <= 2e45.
    """
    if tail not in _TAILS:
        raise ValueError(f"tail must be one of {sorted(_TAILS)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    loss = L.ext().distill_loss(logits, teacher_ids, teacher_logprobs, float(temp), _TAILS[tail], weights,
                                _REDUCTIONS[reduction])
    return loss.view(logits.shape[:-1]) if reduction == "none" else loss
