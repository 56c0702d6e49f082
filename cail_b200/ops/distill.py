"""Distillation from a teacher's top logits."""
from __future__ import annotations

from typing import Optional

import torch

from . import ext

_REDUCTIONS = {"mean": 1, "sum": 0, "none": -1}


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                 targets: Optional[torch.Tensor] = None, temperature: float = 1.0, hard_weight: float = 0.0,
                 reduction: str = "mean") -> torch.Tensor:
    """A student's loss against a teacher's K top logits, float32.

    Per row, with tau = ``temperature``, w = ``hard_weight``, p = softmax of
    ``teacher_logits`` / tau over the row's K entries and q = softmax of
    ``logits`` / tau over the whole vocabulary:

        (1 - w) tau^2 sum_k p_k (log p_k - log q[teacher_ids[k]])
        + w cross_entropy(logits, targets)

    logits are [N, V] (float32, bfloat16 or float16), teacher_ids (int32 or
    int64) and teacher_logits [N, K] with K up to 1024.  A teacher entry whose
    id is outside [0, V) is left out (pad with -1); a row without entries has no
    first term; an id that comes twice counts twice.  With ``targets`` [N], a
    row whose target is outside [0, V) is left out altogether (pad with -100):
    its loss and gradient are 0 and its logits are not read.  ``hard_weight``
    above 0 needs targets.  ``reduction`` is "mean" over the rows that count (0
    if none does), "sum", or "none" ([N]).

    A row whose teacher entries hold NaN or plus infinity, or minus infinity
    alone, has a loss and a gradient of NaN.

    The gradient flows to ``logits``.  Softmax statistics and sums are 32-bit,
    of differences from the row's largest values, so logits may lie around any
    level and be masked by any value; the sum over rows is 64-bit, in a fixed
    order: the same inputs give the same bits.
    """
    try:
        mean = _REDUCTIONS[reduction]
    except KeyError:
        raise ValueError(f"distill_loss: unknown reduction {reduction!r}") from None
    return ext.get_ops().distill_loss(logits, teacher_ids, teacher_logits, targets, temperature, hard_weight, mean)
