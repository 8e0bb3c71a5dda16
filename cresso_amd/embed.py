"""Embedding lookup with a scale, and the dense gradient of its table
(kernels: csrc/embedding.hip)."""

from __future__ import annotations

import torch

from . import _native

WHAT = "embedding"


def _check_ids(what: str, ids: torch.Tensor) -> torch.Tensor:
    _native.require(ids.dtype in (torch.int32, torch.int64), what, f"ids must be int32 or int64, not {ids.dtype}")
    return ids.contiguous()


def _forward(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    rows, width = weight.shape
    weight, stride = _native.rows_of(weight)
    out = torch.empty((*ids.shape, width), dtype=weight.dtype, device=weight.device)
    if out.numel():
        lib = _native.load()
        _native.call(lib.cresso_embedding_forward, WHAT, weight.device, ids.data_ptr(), ids.element_size(), ids.numel(),
                     weight.data_ptr(), rows, width, stride, _native.DTYPE_CODE[weight.dtype], scale, out.data_ptr())
    return out


def embedding_grad(ids: torch.Tensor, grad: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient [rows, width] of a table from the gradient [*ids.shape, width]
    of :func:`embedding`'s output.

    Row v is scale times the sum of grad[t] over the tokens with ids[t] == v,
    in fp32 and in the tokens' order (the same on every run), rounded once to
    grad's dtype; rows that no id names are zero.
    """
    device = _native.require_gpu(WHAT, ids=ids, grad=grad)
    ids = _check_ids(WHAT, ids)
    _native.require(grad.dtype in _native.ROW_DTYPES, WHAT, f"grad must be fp32, bf16 or fp16, not {grad.dtype}")
    _native.require(grad.ndim == ids.ndim + 1 and grad.shape[:-1] == ids.shape, WHAT,
                    f"grad of shape {tuple(grad.shape)} for ids of shape {tuple(ids.shape)}")
    _native.require(rows >= 0, WHAT, "rows must not be negative")
    width = grad.shape[-1]
    grad, stride = _native.rows_of(grad)
    table = torch.empty((rows, width), dtype=grad.dtype, device=device)
    if table.numel():
        lib, code = _native.load(), _native.DTYPE_CODE[grad.dtype]
        nbytes = lib.cresso_embedding_backward_workspace_bytes(ids.numel(), width, code)
        ws = _native.workspace(nbytes, device)
        _native.call(lib.cresso_embedding_backward, "embedding gradient", device, ids.data_ptr(), ids.element_size(),
                     ids.numel(), grad.data_ptr(), stride, rows, width, code, scale, table.data_ptr(), ws.data_ptr(), nbytes)
    return table


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = weight.shape[0], scale
        return _forward(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return None, embedding_grad(ctx.saved_tensors[0], grad, ctx.rows, ctx.scale), None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids]: rows of a table [rows, width] of fp32, bf16 or fp16.

    ids: int32 or int64 of any shape.  An id outside the table (padding, a
    masked token, another shard's word) gives a row of zeros and takes no
    gradient.  The product with scale is formed in fp32 and rounded once.
    The table's gradient is dense (see :func:`embedding_grad`).
    """
    _native.require_gpu(WHAT, ids=ids, weight=weight)
    ids = _check_ids(WHAT, ids)
    _native.require(weight.ndim == 2, WHAT, f"weight must be [rows, width], not {tuple(weight.shape)}")
    _native.require(weight.dtype in _native.ROW_DTYPES, WHAT, f"weight must be fp32, bf16 or fp16, not {weight.dtype}")
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, float(scale))
    return _forward(ids, weight, float(scale))
