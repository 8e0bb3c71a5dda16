"""Products with a frozen weight in 8-bit floating point, one fp32 scale for
each block of 128 x 128 (kernels: csrc/block_product.hip, host side:
csrc/operators.cpp)."""

from __future__ import annotations

from typing import Tuple

import torch

from . import _native


def block_product(x: torch.Tensor, values: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """x [..., inputs] times the transpose of a weight [outputs, inputs] that is
    held as float8_e4m3fn values and one fp32 scale for each block of 128 x 128
    ([ceil(outputs/128), ceil(inputs/128)]); -> [..., outputs] in x's dtype.

    x (fp32, bf16, fp16) is rounded to e4m3 in the call, with one power of two
    for each row and 128 of its elements: the smallest 2^e with max|x| <= 448 *
    2^e (e >= -117), taken over the finite ones.  An infinity or NaN makes its
    row's outputs NaN; what would round to 2^128 becomes 15/16 of it.  A block
    whose scale is 0 counts as zeros whatever its values are.  Sums are fp32,
    rounded once.

    The weight is frozen: the gradient goes to x alone, as the product of the
    incoming gradient, rounded in the same manner, with the weight.
    """
    try:
        return _native.operators().block_product(x, values, scales)
    except TypeError:
        _native.check_tensors("block_product", x=x, values=values, scales=scales)
        raise


def quantize_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (values, scales) of a weight [outputs, inputs] for :func:`block_product`:
    each block's scale is its largest finite magnitude over 448 (1 for a block
    without any, or below 2^-100), its values are weight / scale rounded to
    e4m3, and what is not finite becomes NaN."""
    try:
        return _native.operators().quantize_blocks(weight)
    except TypeError:
        _native.check_tensors("quantize_blocks", weight=weight)
        raise
