"""Distillation from a teacher's top logits: the loss and its gradient
(kernels: csrc/distill.hip, host side: csrc/operators.cpp)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native


def distill_loss(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                 labels: Optional[torch.Tensor] = None, row_weights: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, mix: float = 1.0, ignore_index: int = -100,
                 reduction: str = "sum") -> torch.Tensor:
    """The loss of student logits [rows, vocabulary] against a teacher's top logits.

        p    = softmax(teacher_logits / temperature)      over the entries that are present
        loss = sum over rows of  w * (mix * temperature^2 * KL(p || softmax(logits / temperature))
                                      + (1 - mix) * cross entropy(logits, label))

    teacher_index, teacher_logits: [rows, entries] (at most 1024); an entry
    whose index is outside the vocabulary (-1) is absent, and a row whose
    entries are all absent (or -inf) has no KL term.  labels: [rows]; a label
    that is ignore_index or outside the vocabulary, and no labels at all, leave
    the cross entropy out.  row_weights: fp32 [rows], 1/rows each where not
    given; a row of weight 0 gives no loss and no gradient whatever it holds,
    and a term whose factor is 0 (mix 1 or 0) nothing either.  Masked logits
    may be any finite number or -inf.
    reduction: "sum" (fp32 scalar) or "none" (fp32 [rows], weighted).

    The gradient goes to the logits alone.  Where the loss is the end of the
    program, :func:`distill_loss_and_grad` gives both in one call,
    without keeping anything for a backward pass.
    """
    if reduction not in ("sum", "none"):
        raise ValueError(f"distill_loss: reduction must be 'sum' or 'none', not {reduction!r}")
    try:
        return _native.operators().distill_loss(logits, teacher_index, teacher_logits, labels, row_weights, temperature, mix,
                                                ignore_index, reduction == "sum")
    except TypeError:
        _check(logits, teacher_index, teacher_logits, labels, row_weights)
        raise


def distill_loss_and_grad(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                          labels: Optional[torch.Tensor] = None, row_weights: Optional[torch.Tensor] = None,
                          temperature: float = 1.0, mix: float = 1.0, ignore_index: int = -100,
                          out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (summed loss, its gradient with respect to the logits) of
    :func:`distill_loss`, for programs that drive the backward pass from the
    logits themselves (``logits.backward(grad)``).  `out`: where the gradient
    goes, rows at any stride; it may be `logits` itself (the same rows at the
    same stride), but share no other memory with the inputs."""
    try:
        return _native.operators().distill_loss_and_grad(logits, teacher_index, teacher_logits, labels, row_weights,
                                                         temperature, mix, ignore_index, out)
    except TypeError:
        _check(logits, teacher_index, teacher_logits, labels, row_weights, out)
        raise


def _check(logits, index, teacher, labels, weights, out=None) -> None:
    _native.check_tensors("distill_loss", logits=logits, teacher_index=index, teacher_logits=teacher, labels=labels,
                          row_weights=weights, out=out)
