"""Embedding lookup with a scale, and the dense gradient of its table
(kernels: csrc/embedding.hip, host side: csrc/operators.cpp)."""

from __future__ import annotations

import torch

from . import _native


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids]: rows of a table [rows, width] of fp32, bf16 or fp16.

    ids: int32 or int64 of any shape.  An id outside the table (padding, a
    masked token, another shard's word) gives a row of zeros and takes no
    gradient.  The product with scale is formed in fp32 and rounded once.
    The table's gradient is dense (see :func:`embedding_grad`).
    """
    try:
        return _native.operators().embedding(ids, weight, scale)
    except TypeError:
        _native.check_tensors("embedding", ids=ids, weight=weight)
        raise


def embedding_grad(ids: torch.Tensor, grad: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient [rows, width] of a table from the gradient [*ids.shape, width]
    of :func:`embedding`'s output.

    Row v is scale times the sum of grad[t] over the tokens with ids[t] == v,
    in fp32 and in the tokens' order (the same on every run), rounded once to
    grad's dtype; rows that no id names are zero.
    """
    try:
        return _native.operators().embedding_grad(ids, grad, rows, scale)
    except TypeError:
        _native.check_tensors("embedding", ids=ids, grad=grad)
        raise
