"""Layer norm on MI355X, over the model's width or over each head's row, with its gradients.

``layer_norm(x, weight, bias, eps)`` normalises the last dimension of x:
y = (x - mean) / sqrt(var + eps) * weight + bias, statistics in fp32 and one
rounding to x's dtype.  weight and bias hold [D] elements, or [G, D] for the
last two dimensions of x: each of the G groups (heads) of a row is normalised
by itself and has its own weights.  x may be bf16, fp16 or fp32 and have any
row stride; weight and bias may have any floating dtype (used in fp32, their
gradients are summed in fp32 in a fixed order).
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _launch


def norm_forward(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, groups: int,
                 eps: float) -> torch.Tensor:
    """Raw launch: y, contiguous."""
    return _launch.native().norm_forward(x, weight, bias, groups, eps)


def norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, groups: int, eps: float,
                  need_dx: bool, need_dw: bool, need_db: bool
                  ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Raw launches: (dx like x, dweight, dbias fp32 [groups * D]); None where not needed."""
    return _launch.native().norm_backward(dy, x, weight, groups, eps, need_dx, need_dw, need_db)


class _LayerNormFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups: int, eps: float):
        y = torch.ops.dwarf.layer_norm_fwd(x, weight, bias, groups, eps)
        ctx.save_for_backward(x, weight)
        ctx.groups, ctx.eps = groups, eps
        ctx.table = None if weight is None else (weight.shape, weight.dtype)
        ctx.bias = None if bias is None else (bias.shape, bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        dx, dw, db = torch.ops.dwarf.layer_norm_bwd(dy, x, weight, ctx.groups, ctx.eps, *need)
        return (dx if need[0] else None, dw.view(ctx.table[0]).to(ctx.table[1]) if need[1] else None,
                db.view(ctx.bias[0]).to(ctx.bias[1]) if need[2] else None, None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of the last dimension; weight and bias [D], or [G, D] over the last two dimensions, or None."""
    if not torch.compiler.is_compiling():
        y = _launch.native().layer_norm(x, weight, bias, eps)
        if y is not None:   # None: fake or wrapped tensors, a mode or a trace
            return y
    groups = _check(x, weight, bias, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFn.apply(x, weight, bias, groups, float(eps))
    return torch.ops.dwarf.layer_norm_fwd(x, weight, bias, groups, float(eps))


def _check(x, weight, bias, eps) -> int:
    """The native call's checks, for compiled and traced calls; returns the groups."""
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last dimension to normalise, got {tuple(x.shape)}")
    groups = 1
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.ndim not in (1, 2) or tuple(t.shape) != tuple(x.shape[x.ndim - t.ndim:]):
            raise ValueError(f"{name} must hold the last one or two dimensions of x {tuple(x.shape)}, got {tuple(t.shape)}")
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating point, got {t.dtype}")
        if t.ndim == 2:
            groups = t.shape[0]
    if weight is not None and bias is not None and weight.shape != bias.shape:
        raise ValueError("weight and bias must share a shape")
    if groups < 1:
        raise ValueError("weight and bias need at least one group")
    _launch.check_dtype("x", x)
    _launch.check_device(x, weight=weight, bias=bias)
    return groups
