"""The norm over a set of gradients, and clipping by it (kernels:
csrc/clip.hip, host side: csrc/operators.cpp)."""

from __future__ import annotations

from typing import Iterable, List, Optional

import torch

from . import _native


def gradient_norm(grads: Iterable[Optional[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm over all elements of `grads` (a tensor, or tensors of fp32, fp64,
    bf16 and fp16, None among them): 2 or infinity.  -> fp32 scalar on their GPU,
    0 for no elements, infinite above fp32's range, NaN with a NaN.  Sums are
    fp64, in the same order on every run; squares of fp64 gradients neither
    overflow nor vanish in them."""
    given = _listed(grads)
    try:
        return _native.operators().gradient_norm(given, _kind("gradient_norm", norm_type))
    except TypeError:
        _check("gradient_norm", given)
        raise


def clip_gradients(grads: Iterable[Optional[torch.Tensor]], max_norm: float, *, norm_type: float = 2.0, grad_scale: float = 1.0,
                   out: Optional[Iterable[Optional[torch.Tensor]]] = None) -> torch.Tensor:
    """Scales `grads` so that their norm is at most `max_norm`; -> the norm before.

        norm = |grad_scale| * gradient_norm(grads, norm_type)
        g   <- g * grad_scale * (max_norm / norm  where norm is finite and above max_norm, else 1)

    in fp64, rounded to the gradient's type.  grad_scale undoes a loss scale (1/65536
    for a loss times 65536).  A norm that is infinite or NaN clips nothing: the
    gradients, times grad_scale, stay as they are.  The norm that counts is the
    fp64 one; what is returned is rounded to fp32, so that a norm above fp32's
    range clips but returns infinity.  Nothing waits for the GPU, and where
    nothing changes nothing is written.

    out: where the results go instead, a tensor for each gradient of its shape
    and its type, or fp32 for gradients of 16 bits (then nothing is rounded to 16
    bits a second time); it is always written.  Memory that is written may
    belong to one gradient only (ValueError otherwise; slices that interleave are
    taken as columns of the same rows), but a gradient may be its own output.
    Outside torch.no_grad() it may be no leaf that requires a gradient
    (RuntimeError): these are gradients, not the parameters that have them.
    :meth:`CRESSO5.clip_gradients` takes an optimizer's gradients.
    """
    given, to = _listed(grads), None if out is None else _listed(out)
    try:
        return _native.operators().clip_gradients(given, max_norm, _kind("clip_gradients", norm_type), grad_scale, to)
    except TypeError:
        _check("clip_gradients", given, to or ())
        raise


def _listed(tensors) -> List[Optional[torch.Tensor]]:
    return [tensors] if torch.is_tensor(tensors) else list(tensors)


def _kind(what: str, norm_type: float) -> int:
    kind = {2.0: _native.NORM_2, float("inf"): _native.NORM_MAX}.get(norm_type)
    if kind is None:
        raise ValueError(f"{what}: norm_type must be 2 or infinity, not {norm_type!r}")
    return kind


def _check(what: str, grads, out=()) -> None:
    for t in grads:
        _native.check_tensors(what, gradient=t)
    for t in out:
        _native.check_tensors(what, out=t)
