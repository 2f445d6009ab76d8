"""Layer norm and RMS norm on MI355X, over the model's width or over each head's row, with their gradients.

``layer_norm(x, weight, bias, eps)`` normalises the last dimension of x:
y = (x - mean) / sqrt(var + eps) * weight + bias, statistics in fp32 and one
rounding to x's dtype.  weight and bias hold [D] elements, or [G, D] for the
last two dimensions of x: each of the G groups (heads) of a row is normalised
by itself and has its own weights.  x may be bf16, fp16 or fp32 and have any
row stride; weight and bias may have any floating dtype (used in fp32, their
gradients are summed in fp32 in a fixed order).

``rms_norm(x, weight, residual=residual)`` adds the residual stream on the way:
s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight.  The stream may be fp32
beside rows of 16 bits.  ``rms_norm_fp8`` gives the rows in e4m3 with a scale
for each, for products in 8 bits behind the norm.
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
    if not 0 <= eps < math.inf:   # comparisons alone: where shapes are dynamic a trace has eps as a symbol
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


def rms_forward(x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None, groups: int, eps: float,
                eights: bool) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Raw launch: (y, contiguous, of x's dtype or e4m3; the sum, with a residual; the rows' scales, in 8 bits)."""
    return _launch.native().rms_forward(x, weight, residual, groups, eps, eights)


def rms_backward(dy: torch.Tensor, dsum: torch.Tensor | None, stream: torch.Tensor, weight: torch.Tensor | None,
                 groups: int, eps: float, need_dx: bool, need_dr: bool, need_dw: bool
                 ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Raw launches: (dx of dy's dtype, dresidual of the stream's, dweight fp32 [groups * D]); None where not needed.
    One tensor is both dx and dresidual where the dtypes are the same."""
    return _launch.native().rms_backward(dy, dsum, stream, weight, groups, eps, need_dx, need_dr, need_dw)


class _RmsNormFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, x, weight, residual, groups: int, eps: float):
        ctx.set_materialize_grads(False)
        y, total = torch.ops.dwarf.rms_norm_fwd(x, weight, residual, groups, eps)
        ctx.save_for_backward(x if residual is None else total, weight)
        ctx.groups, ctx.eps, ctx.added, ctx.dtype = groups, eps, residual is not None, x.dtype
        ctx.table = None if weight is None else (weight.shape, weight.dtype)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        stream, weight = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if dy is None and dsum is None:
            return None, None, None, None, None
        if dy is None:   # the sum alone was used
            dy = torch.zeros_like(stream, dtype=ctx.dtype)
        dx, dr, dw = torch.ops.dwarf.rms_norm_bwd(dy.to(ctx.dtype), dsum, stream, weight, ctx.groups, ctx.eps, need[0],
                                                  need[2], need[1])
        return (dx if need[0] else None, dw.view(ctx.table[0]).to(ctx.table[1]) if need[1] else None,
                dr if need[2] else None, None, None)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-5):
    """RMS norm of the last dimension; weight [D], or [G, D] over the last two dimensions, or None.

    With a ``residual`` (x's shape; x's dtype, or fp32) the norm is taken of s = x + residual, rounded to residual's
    dtype, and (y, s) is returned: s is the residual stream that goes on.  y has x's dtype.  The norm is that of s as
    returned, and so are the gradients, which come from s and are what both x and residual receive."""
    if not torch.compiler.is_compiling():
        done = _launch.native().rms_norm(x, weight, residual, eps)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    groups = _check_rms(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return _RmsNormFn.apply(x, weight, residual, groups, float(eps))
    y, total = torch.ops.dwarf.rms_norm_fwd(x, weight, residual, groups, float(eps))
    return y if residual is None else (y, total)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
                 eps: float = 1e-5):
    """``rms_norm`` with its rows in 8 bits: (q, scale), with a residual (q, scale, s); y is q * scale.

    q is float8_e4m3fn of x's shape, scale fp32 [..., 1] = max|y| / 448 of the row (of each group's row), at least the
    smallest normal fp32.  y is rounded once, to q.  A row that is not finite holds NaN where its input is not finite.
    No gradients."""
    if not torch.compiler.is_compiling():
        done = _launch.native().rms_norm_fp8(x, weight, residual, eps)
        if done is not None:
            return done
    groups = _check_rms(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradients: call it under torch.no_grad(), or rms_norm")
    q, scale, total = torch.ops.dwarf.rms_norm_fp8(x, weight, residual, groups, float(eps))
    return (q, scale) if residual is None else (q, scale, total)


def _check_rms(x, weight, residual, eps) -> int:
    """The native call's checks, for compiled and traced calls; returns the groups."""
    groups = _check(x, weight, None, eps)
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} and its dtype {x.dtype} or fp32, got "
                         f"{tuple(residual.shape)} {residual.dtype}")
    _launch.check_device(x, residual=residual)
    return groups
