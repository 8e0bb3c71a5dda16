"""The seam between two blocks of a network in one operator: the norm after a
block, its gate, the scaled residual and the norm before the next block
(kernels: csrc/residual_norm.hip, host side: csrc/operators.cpp)."""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _native

GATE_ACT = {"none": 0, "sigmoid": 1, "tanh": 2}


def residual_norm(residual: torch.Tensor, update: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None,
                  gate_act: str = "none", post_weight: Optional[torch.Tensor] = None,
                  pre_weight: Optional[torch.Tensor] = None, residual_scale: Union[float, torch.Tensor] = 1.0,
                  eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """-> (out, normed) with

        out    = residual_scale * residual + act(gate) * (update * rms(update) * post_weight)
        normed = out * rms(out) * pre_weight,            rms(x) = 1 / sqrt(mean(x^2) + eps)

    over the last dimension (at most 16384).  Every part but the residual may
    be left out: without `update` there is no gate and no norm after it;
    without `post_weight` the update is taken as it is; without `pre_weight`
    `normed` is None.

    residual, update: one shape and dtype (fp32, bf16, fp16).  gate: (width,),
    or the leading dimensions of the rows followed by ones, as (batch, 1,
    width), or an element each; gate_act: "none", "sigmoid" or "tanh".
    residual_scale: a number or a vector (width,).  Vectors and gates are of
    the rows' dtype or fp32, and so are their gradients.  Everything is
    computed in fp32 and rounded once; `normed` is formed from the unrounded
    `out`.
    """
    act = GATE_ACT.get(gate_act)
    if act is None:
        raise ValueError(f"residual_norm: gate_act must be one of {sorted(GATE_ACT)}, not {gate_act!r}")
    vec, scale = (residual_scale, 1.0) if torch.is_tensor(residual_scale) else (None, residual_scale)
    try:
        return _native.operators().residual_norm(residual, update, gate, act, post_weight, pre_weight, vec, scale, eps)
    except TypeError:
        _native.check_tensors("residual_norm", residual=residual, update=update, gate=gate, post_weight=post_weight,
                              pre_weight=pre_weight)
        raise
