"""The seam between two blocks of a network in one operator: the norm after a
block, its gate, the scaled residual and the norm before the next block
(kernels: csrc/residual_norm.hip)."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _native

WHAT = "residual_norm"
GATE_ACT = {"none": 0, "sigmoid": 1, "tanh": 2}


def _gate_rows(gate: torch.Tensor, like: torch.Tensor) -> int:
    """Rows of `like` for each row of a gate of shape (width,) or (leading dims of like, 1, ..., 1, width)."""
    lead, width = like.shape[:-1], like.shape[-1]
    if gate.ndim == 1 and gate.shape[0] == width:
        return max(1, like.numel() // max(1, width))
    ok = gate.ndim == like.ndim and gate.shape[-1] == width
    k = 0
    if ok:
        while k < len(lead) and gate.shape[k] == lead[k]:
            k += 1
        ok = all(n == 1 for n in gate.shape[k:-1])
    _native.require(ok, WHAT, f"gate of shape {tuple(gate.shape)} for rows of shape {tuple(like.shape)}: it must be "
                              f"(width,) or have the rows' own leading dimensions and then ones")
    rows = 1
    for n in lead[k:]:
        rows *= n
    return max(1, rows)


def _vector(name: str, v: Optional[torch.Tensor], like: torch.Tensor) -> Optional[torch.Tensor]:
    if v is None:
        return None
    _native.require(v.dtype in (torch.float32, like.dtype), WHAT, f"{name} must be fp32 or {like.dtype}, not {v.dtype}")
    return v


def _weight(name: str, v: Optional[torch.Tensor], like: torch.Tensor) -> Optional[torch.Tensor]:
    v = _vector(name, v, like)
    if v is not None:
        _native.require(v.shape == like.shape[-1:], WHAT,
                        f"{name} of shape {tuple(v.shape)} for a width of {like.shape[-1]}")
        v = v.contiguous()
    return v


def _fill(residual, update, gate, post, pre, scale_vec, scale, eps, act, rows_per_gate):
    """-> descriptor, what it points to (to be kept until the call)."""
    d = _native.ResidualNormDesc()
    width = residual.shape[-1]
    h, d.residual_stride = _native.rows_of(residual)
    keep = [h]
    d.residual, d.width, d.rows = h.data_ptr(), width, residual.numel() // width
    d.dtype = _native.DTYPE_CODE[residual.dtype]
    if update is not None:
        y, d.update_stride = _native.rows_of(update)
        d.update = y.data_ptr()
        keep.append(y)
    if gate is not None:
        g = gate.contiguous()
        d.gate, d.gate_stride, d.gate_dtype, d.act = g.data_ptr(), width, _native.DTYPE_CODE[g.dtype], act
        keep.append(g)
    d.rows_per_gate = rows_per_gate
    for name, v in (("post", post), ("pre", pre), ("scale", scale_vec)):
        if v is not None:
            setattr(d, "scale_vec" if name == "scale" else name, v.data_ptr())
            setattr(d, name + "_dtype", _native.DTYPE_CODE[v.dtype])
    d.scale, d.eps = scale, eps
    return d, keep


def _forward(residual, update, gate, post, pre, scale_vec, scale, eps, act, rows_per_gate, stats):
    out = torch.empty(residual.shape, dtype=residual.dtype, device=residual.device)
    normed = torch.empty_like(out) if pre is not None else None
    if out.numel():
        d, keep = _fill(residual, update, gate, post, pre, scale_vec, scale, eps, act, rows_per_gate)
        d.out = out.data_ptr()
        if normed is not None:
            d.normed = normed.data_ptr()
        if stats is not None:
            d.stats = stats.data_ptr()
        _native.call(_native.load().cresso_residual_norm_forward, WHAT, residual.device, ctypes.byref(d))
    return out, normed


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, update, gate, post, pre, scale_vec, scale, eps, act, rows_per_gate):
        rows = residual.numel() // max(1, residual.shape[-1])
        stats = torch.empty((rows, 2), dtype=torch.float32, device=residual.device)
        out, normed = _forward(residual, update, gate, post, pre, scale_vec, scale, eps, act, rows_per_gate, stats)
        ctx.save_for_backward(residual, update, gate, post, pre, scale_vec, stats)
        ctx.rest = (scale, eps, act, rows_per_gate)
        ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_normed):
        *inputs, stats = ctx.saved_tensors
        if d_out is None and d_normed is None:
            return (None,) * 10
        residual = inputs[0]
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and ctx.needs_input_grad[i] else None
                 for i, t in enumerate(inputs)]
        if not residual.numel():
            for g in grads:
                if g is not None:
                    g.zero_()
            return (*grads, None, None, None, None)
        d, keep = _fill(*inputs, *ctx.rest)
        d.stats = stats.data_ptr()
        for name, g in (("d_out", d_out), ("d_normed", d_normed)):
            if g is not None:
                t, stride = _native.rows_of(g)
                keep.append(t)
                setattr(d, name, t.data_ptr())
                setattr(d, name + "_stride", stride)
        for name, g in zip(("d_residual", "d_update", "d_gate", "d_post", "d_pre", "d_scale"), grads):
            if g is not None:
                setattr(d, name, g.data_ptr())
        lib = _native.load()
        nbytes = lib.cresso_residual_norm_backward_workspace_bytes(ctypes.byref(d))
        ws = _native.workspace(nbytes, residual.device)
        _native.call(lib.cresso_residual_norm_backward, "residual_norm gradient", residual.device, ctypes.byref(d),
                     ws.data_ptr(), nbytes)
        return (*grads, None, None, None, None)


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
    width), or an element each.  residual_scale: a number or a vector (width,).
    Vectors and gates are of the rows' dtype or fp32, and so are their
    gradients.  Everything is computed in fp32 and rounded once; `normed` is
    formed from the unrounded `out`.
    """
    scale_vec = residual_scale if torch.is_tensor(residual_scale) else None
    _native.require_gpu(WHAT, residual=residual, update=update, gate=gate, post_weight=post_weight, pre_weight=pre_weight,
                        residual_scale=scale_vec)
    _native.require(residual.dtype in _native.ROW_DTYPES, WHAT, f"residual must be fp32, bf16 or fp16, not {residual.dtype}")
    _native.require(residual.ndim >= 1 and residual.shape[-1] >= 1, WHAT, "the last dimension must not be empty")
    _native.require(residual.shape[-1] <= 16384, WHAT, f"width {residual.shape[-1]} above 16384")
    _native.require(gate_act in GATE_ACT, WHAT, f"gate_act must be one of {sorted(GATE_ACT)}, not {gate_act!r}")
    _native.require(eps > 0.0, WHAT, "eps must be positive")
    rows_per_gate = 1
    if update is not None:
        _native.require(update.shape == residual.shape and update.dtype == residual.dtype, WHAT,
                        f"update is {update.dtype} {tuple(update.shape)}, residual {residual.dtype} {tuple(residual.shape)}")
    else:
        _native.require(gate is None and post_weight is None, WHAT, "a gate or post_weight needs an update")
    if gate is not None:
        gate = _vector("gate", gate, residual)
        rows_per_gate = _gate_rows(gate, residual)
    post, pre = _weight("post_weight", post_weight, residual), _weight("pre_weight", pre_weight, residual)
    scale_vec = _weight("residual_scale", scale_vec, residual)
    args = (residual, update, gate, post, pre, scale_vec, 1.0 if scale_vec is not None else float(residual_scale),
            float(eps), GATE_ACT[gate_act], rows_per_gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:6]):
        return _ResidualNorm.apply(*args)
    return _forward(*args, None)
