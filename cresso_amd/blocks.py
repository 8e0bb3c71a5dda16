"""Products with a frozen weight in 8-bit floating point, one fp32 scale for
each block of 128 x 128 (kernels: csrc/block_product.hip)."""

from __future__ import annotations

from typing import Tuple

import torch

from . import _native

WHAT = "block_product"
BLOCK = 128


def _check_weight(values: torch.Tensor, scales: torch.Tensor) -> None:
    _native.require(values.ndim == 2 and values.dtype == torch.float8_e4m3fn, WHAT,
                    f"values must be float8_e4m3fn [outputs, inputs], not {values.dtype} {tuple(values.shape)}")
    blocks = tuple(-(-n // BLOCK) for n in values.shape)
    _native.require(scales.dtype == torch.float32 and tuple(scales.shape) == blocks, WHAT,
                    f"scales must be fp32 {blocks}, not {scales.dtype} {tuple(scales.shape)}")


def _product(x: torch.Tensor, values: torch.Tensor, scales: torch.Tensor, turned: bool) -> torch.Tensor:
    depth, cols = (values.shape[0], values.shape[1]) if turned else (values.shape[1], values.shape[0])
    out = torch.empty((*x.shape[:-1], cols), dtype=x.dtype, device=x.device)
    if out.numel():
        rows = out.numel() // cols
        x, x_stride = _native.rows_of(x)
        values, w_stride = _native.rows_of(values)
        scales = scales.contiguous()
        lib = _native.load()
        nbytes = lib.cresso_block_product_workspace_bytes(rows, cols, depth, values.data_ptr(), w_stride, turned)
        ws = _native.workspace(nbytes, x.device)
        _native.call(lib.cresso_block_product, WHAT, x.device, x.data_ptr(), x_stride, _native.DTYPE_CODE[x.dtype], rows,
                     cols, depth, values.data_ptr(), w_stride, scales.data_ptr(), scales.shape[1], turned, out.data_ptr(),
                     ws.data_ptr(), nbytes)
    return out


class _BlockProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, scales):
        ctx.save_for_backward(values, scales)
        return _product(x, values, scales, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        values, scales = ctx.saved_tensors
        return _product(grad, values, scales, True), None, None


def block_product(x: torch.Tensor, values: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """x [..., inputs] times the transpose of a weight [outputs, inputs] that is
    held as float8_e4m3fn values and one fp32 scale for each block of 128 x 128
    ([ceil(outputs/128), ceil(inputs/128)]); -> [..., outputs] in x's dtype.

    x (fp32, bf16, fp16) is rounded to e4m3 in the call, with one power of two
    for each row and 128 of its elements: the smallest 2^e with max|x| <= 448 *
    2^e (e >= -117), taken over the finite ones.  An infinity or NaN makes its row's
    outputs NaN; what would round to 2^128 becomes 15/16 of it.  Sums are fp32, rounded once.

    The weight is frozen: the gradient goes to x alone, as the product of the
    incoming gradient, rounded in the same manner, with the weight.
    """
    _native.require_gpu(WHAT, x=x, values=values, scales=scales)
    _check_weight(values, scales)
    _native.require(x.dtype in _native.ROW_DTYPES, WHAT, f"x must be fp32, bf16 or fp16, not {x.dtype}")
    _native.require(x.ndim >= 1 and x.shape[-1] == values.shape[1], WHAT,
                    f"x of shape {tuple(x.shape)} for a weight of {values.shape[1]} inputs")
    if x.requires_grad and torch.is_grad_enabled():
        return _BlockProduct.apply(x, values, scales)
    return _product(x, values, scales, False)


@torch.no_grad()
def quantize_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (values, scales) of a weight [outputs, inputs] for :func:`block_product`:
    each block's scale is its largest finite magnitude over 448 (1 for a block
    without any, or below 2^-100), its values are weight / scale rounded to
    e4m3, and what is not finite becomes NaN."""
    device = _native.require_gpu(WHAT, weight=weight)
    _native.require(weight.ndim == 2, WHAT, f"weight must be [outputs, inputs], not {tuple(weight.shape)}")
    _native.require(weight.dtype in _native.ROW_DTYPES, WHAT, f"weight must be fp32, bf16 or fp16, not {weight.dtype}")
    rows, cols = weight.shape
    values = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty((-(-rows // BLOCK), -(-cols // BLOCK)), dtype=torch.float32, device=device)
    if values.numel():
        w, stride = _native.rows_of(weight)
        _native.call(_native.load().cresso_block_quantize, "quantize_blocks", device, w.data_ptr(), stride,
                     _native.DTYPE_CODE[w.dtype], rows, cols, values.data_ptr(), scales.data_ptr())
    return values, scales
