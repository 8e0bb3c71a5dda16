"""Distillation from a teacher's top logits: the loss and its gradient
(kernels: csrc/distill.hip)."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _native

WHAT = "distill_loss"
MAX_TOP = 1024


def _fill(logits, index, teacher, labels, weights, temperature, mix, ignore_index):
    """-> descriptor, what it points to (to be kept until the call)."""
    d = _native.DistillDesc()
    z, d.logits_stride = _native.rows_of(logits)
    i, d.index_stride = _native.rows_of(index)
    a, d.teacher_stride = _native.rows_of(teacher)
    d.logits, d.index, d.teacher = z.data_ptr(), i.data_ptr(), a.data_ptr()
    d.rows, d.vocab = logits.shape
    d.top = index.shape[1]
    d.dtype, d.teacher_dtype = _native.DTYPE_CODE[logits.dtype], _native.DTYPE_CODE[teacher.dtype]
    d.index_bytes = index.element_size()
    keep = [z, i, a]
    if labels is not None:
        labels = labels.contiguous()
        d.labels, d.label_bytes = labels.data_ptr(), labels.element_size()
        keep.append(labels)
    if weights is not None:
        weights = weights.contiguous()
        d.weights = weights.data_ptr()
        keep.append(weights)
    d.weight = 1.0 / max(1, d.rows)
    d.temperature, d.mix, d.ignore_index = temperature, mix, ignore_index
    return d, keep


def _check(logits, index, teacher, labels, weights, temperature, mix):
    _native.require_gpu(WHAT, logits=logits, teacher_index=index, teacher_logits=teacher, labels=labels, row_weights=weights)
    _native.require(logits.ndim == 2 and logits.shape[1] >= 1, WHAT, f"logits must be [rows, vocabulary], not {tuple(logits.shape)}")
    rows = logits.shape[0]
    _native.require(index.ndim == 2 and index.shape[0] == rows and teacher.shape == index.shape, WHAT,
                    f"teacher_index {tuple(index.shape)} and teacher_logits {tuple(teacher.shape)} must both be "
                    f"[{rows}, entries]")
    _native.require(index.shape[1] <= MAX_TOP, WHAT, f"{index.shape[1]} teacher entries a row: at most {MAX_TOP}")
    for name, t in (("logits", logits), ("teacher_logits", teacher)):
        _native.require(t.dtype in _native.ROW_DTYPES, WHAT, f"{name} must be fp32, bf16 or fp16, not {t.dtype}")
    for name, t in (("teacher_index", index), ("labels", labels)):
        _native.require(t is None or t.dtype in (torch.int32, torch.int64), WHAT, f"{name} must be int32 or int64")
    _native.require(labels is None or labels.shape == (rows,), WHAT, f"labels must be [{rows}]")
    _native.require(weights is None or (weights.shape == (rows,) and weights.dtype == torch.float32), WHAT,
                    f"row_weights must be fp32 [{rows}]")
    _native.require(temperature > 0.0, WHAT, "temperature must be positive")
    _native.require(0.0 <= mix <= 1.0, WHAT, "mix must be within 0..1")


def _loss(args, total: bool, stats=None, grad=None):
    """-> rows' losses, their sum or None."""
    logits = args[0]
    rows = logits.shape[0]
    losses = torch.empty(rows, dtype=torch.float32, device=logits.device)
    summed = torch.empty((), dtype=torch.float32, device=logits.device) if total else None
    d, keep = _fill(*args)
    d.loss = losses.data_ptr()
    if total:
        d.total = summed.data_ptr()
    if stats is not None:
        d.stats = stats.data_ptr()
    if grad is not None:
        d.grad, d.grad_stride = grad.data_ptr(), grad.stride(0)
    _native.call(_native.load().cresso_distill_loss, WHAT, logits.device, ctypes.byref(d))
    return losses, summed


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, labels, weights, temperature, mix, ignore_index, total):
        stats = torch.empty((logits.shape[0], 3), dtype=torch.float32, device=logits.device)
        losses, summed = _loss((logits, index, teacher, labels, weights, temperature, mix, ignore_index), total, stats)
        ctx.save_for_backward(logits, index, teacher, labels, weights, stats)
        ctx.rest = (temperature, mix, ignore_index)
        return summed if total else losses

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        *inputs, stats = ctx.saved_tensors
        logits = inputs[0]
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if grad.numel():
            d, keep = _fill(*inputs, *ctx.rest)
            d.stats, d.d_loss = stats.data_ptr(), d_loss.data_ptr()
            d.d_loss_stride = d_loss.stride(0) if d_loss.ndim else 0
            d.grad, d.grad_stride = grad.data_ptr(), grad.shape[1]
            _native.call(_native.load().cresso_distill_backward, "distill_loss gradient", logits.device, ctypes.byref(d))
        return (grad,) + (None,) * 8


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
    given; a row of weight 0 gives no loss and no gradient whatever it holds.
    reduction: "sum" (fp32 scalar) or "none" (fp32 [rows], weighted).

    The gradient goes to the logits alone.  Where the loss is the end of the
    program, :func:`distill_loss_and_grad` gives both in one pass.
    """
    _check(logits, teacher_index, teacher_logits, labels, row_weights, temperature, mix)
    _native.require(reduction in ("sum", "none"), WHAT, f"reduction must be 'sum' or 'none', not {reduction!r}")
    args = (logits, teacher_index, teacher_logits, labels, row_weights, float(temperature), float(mix), int(ignore_index))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(*args, reduction == "sum")
    losses, summed = _loss(args, reduction == "sum")
    return losses if summed is None else summed


@torch.no_grad()
def distill_loss_and_grad(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                          labels: Optional[torch.Tensor] = None, row_weights: Optional[torch.Tensor] = None,
                          temperature: float = 1.0, mix: float = 1.0, ignore_index: int = -100,
                          out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (summed loss, its gradient with respect to the logits) of
    :func:`distill_loss`, for programs that drive the backward pass from the
    logits themselves (``logits.backward(grad)``).  `out`: where the gradient
    goes, rows at any stride; it may be `logits` itself."""
    _check(logits, teacher_index, teacher_logits, labels, row_weights, temperature, mix)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    else:
        _native.require_gpu(WHAT, logits=logits, out=out)
        _native.require(out.shape == logits.shape and out.dtype == logits.dtype, WHAT,
                        f"out is {out.dtype} {tuple(out.shape)}, logits {logits.dtype} {tuple(logits.shape)}")
        _native.require(out.stride(1) == 1 and (out.shape[0] < 2 or out.stride(0) >= out.shape[1]), WHAT,
                        "out must hold each row in one piece")
    args = (logits, teacher_index, teacher_logits, labels, row_weights, float(temperature), float(mix), int(ignore_index))
    _, total = _loss(args, True, grad=out)
    return total, out
