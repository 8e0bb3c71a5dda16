"""Layers of experts: the router, the rows' way to the experts and back, and the
products with each expert's matrix (kernels: csrc/routing.hip,
csrc/expert_rows.hip, csrc/expert_product.hpp; host side: csrc/operators.cpp).

    weights, routing = route_experts(logits, top=2)              # which experts take each token
    rows = dispatch_rows(x, routing)                             # the tokens' rows, sorted by expert
    rows = expert_product(rows, weight, routing.offsets)         # each with its expert's matrix
    y = combine_rows(rows, routing, weights)                     # back, summed over each token's experts
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native


class Routing(NamedTuple):
    """Where tokens go, int32 on their GPU.  A slot is token * top + entry.

    experts [tokens, top]: each token's experts, -1 for absent ones (they come
    last); order [tokens * top]: the slots sorted by expert, those of one expert
    in their own order, absent ones last; places [tokens, top]: each slot's row
    in that order; offsets [experts + 1]: where each expert's rows begin, and the
    last's end.
    """

    experts: torch.Tensor
    order: torch.Tensor
    places: torch.Tensor
    offsets: torch.Tensor


_SCORES = {"softmax": _native.SCORE_SOFTMAX, "sigmoid": _native.SCORE_SIGMOID}


def route_experts(logits: torch.Tensor, top: int, *, score: str = "softmax", normalize: bool = True, scale: float = 1.0,
                  bias: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Routing]:
    """-> (weights [tokens, top] in fp32, :class:`Routing`) from the router's logits
    [tokens, experts] (fp32, bf16, fp16; at most 1024 experts and 32 a token).

    A token takes the `top` experts of the largest logit + bias (fp32), the lowest
    expert where they are equal; NaN counts as the largest, and -inf is never
    taken: where fewer are left the last entries are absent, with weight 0.
    The bias is added to the logit, not to its softmax or sigmoid: a bias that was
    trained beside those chooses other experts here.  Their weights come from the
    logits without the bias (which balances the load and takes no gradient):

        softmax   scale * softmax(logits), over all experts or, with `normalize`, over the chosen ones
        sigmoid   scale * sigmoid(logits), with `normalize` divided by the chosen ones' sum

    in fp32.  The gradient goes from the weights to the logits.
    """
    if score not in _SCORES:
        raise ValueError(f"route_experts: score must be one of {sorted(_SCORES)}, not {score!r}")
    try:
        weights, *routing = _native.operators().route_experts(logits, top, _SCORES[score], normalize, scale, bias)
    except TypeError:
        _native.check_tensors("route_experts", logits=logits, bias=bias)
        raise
    return weights, Routing(*routing)


def dispatch_rows(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """-> rows [tokens * top, width]: each token's row of x [tokens, width] (fp32,
    bf16, fp16) once for each of its experts, sorted by expert; zeros for absent
    ones, behind the last expert's rows.  The gradient of a token is the sum of
    its rows' gradients, in fp32, rounded once."""
    try:
        return _native.operators().dispatch_rows(x, routing.experts, routing.places)
    except (TypeError, AttributeError):
        _check_routing("dispatch_rows", routing, x=x)
        raise


def combine_rows(rows: torch.Tensor, routing: Routing, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """-> [tokens, width]: the sum of each token's rows [tokens * top, width], times
    `weights` (fp32 [tokens, top]; 1 where not given), in fp32, rounded once.
    Absent experts add nothing, whatever their rows hold, and take gradients of
    zero.  The gradient goes to the rows and the weights."""
    try:
        return _native.operators().combine_rows(rows, routing.experts, routing.places, weights)
    except (TypeError, AttributeError):
        _check_routing("combine_rows", routing, rows=rows, weights=weights)
        raise


def expert_product(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Rows of x [rows, inputs] times the transpose of their expert's matrix:
    -> [rows, outputs] in x's dtype.

    weight: [experts, outputs, inputs] of x's dtype (fp32, bf16, fp16), as one
    parameter; a transposed view of [experts, inputs, outputs] is taken where it
    lies too.  offsets: int32 [experts + 1] on the GPU, within 0..rows and not
    falling: rows offsets[e] to offsets[e + 1] are expert e's, any number of
    them.  Rows outside offsets[0]..offsets[-1] give zeros and take gradients of
    zero, whatever they hold; an expert without rows takes one too.  Sums are
    fp32, rounded once.
    """
    try:
        return _native.operators().expert_product(x, weight, offsets)
    except TypeError:
        _native.check_tensors("expert_product", x=x, weight=weight, offsets=offsets)
        raise


def _check_routing(what: str, routing, **given) -> None:
    _native.check_tensors(what, **given)
    for k in ("experts", "places"):
        t = getattr(routing, k, None)
        if not torch.is_tensor(t):
            raise ValueError(f"{what}: routing must be what route_experts returns, not {type(routing).__name__}")
