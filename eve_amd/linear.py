"""A linear layer with its epilogue fused (eve_linear_fwd / eve_linear_bwd): the products around the encoder's attention and
the residual branch that follows the second one (reference models/multiway_transformer.py:104-106, :129-130, :341), one pass
each instead of the product, the layer scale, the DropPath product and the sum.  No CPU fallback.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import ops


def _rows(x, weight, bias, gamma, row_scale, residual):
    """The tensors as the kernels take them, contiguous and with the leading dimensions in one, and the rows of a sample."""
    N, K = weight.shape
    rows = math.prod(x.shape[:-1])
    small = [None if t is None else t.contiguous() for t in (bias, gamma, row_scale)]
    res2 = None if residual is None else residual.contiguous().view(rows, N)
    per = max(1, rows // max(1, x.shape[0])) if row_scale is not None else 1
    return (x.contiguous().view(rows, K), weight.contiguous(), *small, res2, per)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gamma, row_scale, residual, act):  # type: ignore[override]
        x2, weight, bias, gamma, row_scale, res2, per = _rows(x, weight, bias, gamma, row_scale, residual)
        need = ctx.needs_input_grad
        product = need[0] or need[1] or need[2]
        y, z = ops.linear_fwd(x2, weight, bias, gamma, row_scale, res2, per, act,
                              save_z=need[3] or (product and act != ops.ACTS["identity"]))
        if product or need[3]:
            ctx.save_for_backward(x2, weight, z, gamma, row_scale)
        ctx.how = (x.shape, per, act)
        return y.view(x.shape[:-1] + (weight.shape[0],))

    @staticmethod
    @ops.once_differentiable
    def backward(ctx, dy):  # type: ignore[override]
        shape, per, act = ctx.how
        need = ctx.needs_input_grad
        dx = dw = db = dg = None
        if need[0] or need[1] or need[2] or need[3]:
            x2, weight, z, gamma, row_scale = ctx.saved_tensors
            dx, dw, db, dg = ops.linear_bwd(dy.contiguous().view(x2.shape[0], weight.shape[0]), x2, weight, z, gamma, row_scale, per, act,
                                            need[:4])
        return None if dx is None else dx.view(shape), dw, db, dg, None, dy if need[5] else None, None


def fused_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "identity",
                 gamma: Optional[Tensor] = None, row_scale: Optional[Tensor] = None,
                 residual: Optional[Tensor] = None) -> Tensor:
    """residual + row_scale * gamma * act(x @ weight.T + bias), differentiable in all but row_scale.

    x [..., K]; weight [N, K]; bias, gamma [N]; row_scale [x.shape[0]], one factor per sample (DropPath's mask / keep
    probability); residual [..., N]; all of one type, float32 or bfloat16.  activation: "identity", "quick_gelu", "gelu" or
    "relu".  Everything after the product works on its float32 accumulator and is rounded once; gradients are summed in a
    fixed order."""
    if activation not in ops.ACTS:
        raise ValueError(f"eve_amd.fused_linear: activation {activation!r} (one of {', '.join(ops.ACTS)})")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"eve_amd.fused_linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not belong together")
    ops._dt(x)
    dtype, device, lead = x.dtype, x.device, x.shape[:-1]
    N = weight.shape[0]
    if max(math.prod(lead), *weight.shape) >= 1 << 31:  # the C calls' sizes are 32-bit
        raise ValueError(f"eve_amd.fused_linear: x {tuple(x.shape)}, weight {tuple(weight.shape)} (2^31 rows or columns and more are not supported)")
    parts = (("weight", weight, weight.shape), ("bias", bias, (N,)), ("gamma", gamma, (N,)), ("row_scale", row_scale, x.shape[:1]),
             ("residual", residual, lead + (N,)))
    elsewhere = "" if not x.is_cuda else None
    for name, t, shape in parts:
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"eve_amd.fused_linear: `{name}` is {t.dtype}, x {dtype}")
        if t.shape != shape:
            raise ValueError(f"eve_amd.fused_linear: `{name}` has shape {tuple(t.shape)}, {tuple(shape)} is needed")
        if t.device != device:
            elsewhere = f", `{name}` on {t.device}"
    if row_scale is not None and x.dim() < 2:
        raise ValueError("eve_amd.fused_linear: row_scale needs samples: x with two dimensions or more")
    if row_scale is not None and row_scale.requires_grad:
        raise ValueError("eve_amd.fused_linear: row_scale is a mask and has no gradient")
    if elsewhere is not None:
        raise RuntimeError(f"eve_amd.fused_linear runs on one MI355X (x on {device}{elsewhere}); no CPU fallback")
    act = ops.ACTS[activation]
    if ops._tracks(x, weight, bias, gamma, residual):
        return _LinearFn.apply(x, weight, bias, gamma, row_scale, residual, act)
    return ops.linear_fwd(*_rows(x, weight, bias, gamma, row_scale, residual), act)[0].view(lead + (N,))
