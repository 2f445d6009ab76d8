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

from . import _launch, _lib


def _strides(x: torch.Tensor, groups: int) -> tuple[int, int] | None:
    """(row stride, group stride) of x as [rows][groups][D]; None where the leading dimensions do not collapse."""
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        return None
    lead = list(zip(x.shape, x.stride()))[:-1]
    inner = 0
    if groups > 1:
        inner = lead.pop()[1]
    lead = [(n, s) for n, s in lead if n != 1]
    for (_, outer), (n, s) in zip(lead, lead[1:]):
        if outer != n * s:
            return None
    return (lead[-1][1] if lead else 0), inner


def _operand(x: torch.Tensor, groups: int) -> tuple[torch.Tensor, tuple[int, int]]:
    s = _strides(x, groups)
    if s is None:
        x = x.contiguous()
        s = _strides(x, groups)
    return x, s


def _table(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.detach().float().contiguous()


def _fill(a: _lib.LayerNormFwdArgs, x: torch.Tensor, groups: int, strides, weight, bias, eps: float) -> None:
    D = x.shape[-1]
    a.rows, a.groups, a.D = x.numel() // (groups * D), groups, D
    a.dtype, a.eps = _launch.DTYPES[x.dtype], eps
    a.x, a.x_stride = x.data_ptr(), strides
    a.weight = None if weight is None else weight.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()


def norm_forward(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, groups: int,
                 eps: float) -> torch.Tensor:
    """Raw launch: y, contiguous."""
    x, strides = _operand(x, groups)
    weight, bias = _table(weight), _table(bias)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    a = _lib.LayerNormFwdArgs()
    _fill(a, x, groups, strides, weight, bias, eps)
    a.y, a.y_stride = y.data_ptr(), (groups * x.shape[-1], x.shape[-1])
    _launch.launch("dwarf_layer_norm_fwd", a, x.device)
    return y


def norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, groups: int, eps: float,
                  need_dx: bool, need_dw: bool, need_db: bool
                  ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Raw launches: (dx like x, dweight, dbias fp32 [groups * D]); None where not needed."""
    x, strides = _operand(x, groups)
    dy, dy_strides = _operand(dy.to(x.dtype), groups)
    weight = _table(weight)
    D = x.shape[-1]
    a = _lib.LayerNormBwdArgs()
    _fill(a.fwd, x, groups, strides, weight, None, eps)
    a.dy, a.dy_stride = dy.data_ptr(), dy_strides
    dx = dw = db = None
    if need_dx:
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        a.dx, a.dx_stride = dx.data_ptr(), (groups * D, D)
    if need_dw:
        dw = torch.empty(groups * D, device=x.device, dtype=torch.float32)
        a.dweight = dw.data_ptr()
    if need_db:
        db = torch.empty(groups * D, device=x.device, dtype=torch.float32)
        a.dbias = db.data_ptr()
    ws = _launch.workspace("dwarf_layer_norm_bwd_workspace_bytes", a, x.device)
    if ws is not None:
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _launch.launch("dwarf_layer_norm_bwd", a, x.device)
    return dx, dw, db


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups: int, eps: float):
        forward = torch.ops.dwarf.layer_norm_fwd if torch.compiler.is_compiling() else norm_forward
        y = forward(x, weight, bias, groups, eps)
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
        if torch.compiler.is_compiling():
            dx, dw, db = torch.ops.dwarf.layer_norm_bwd(dy, x, weight, ctx.groups, ctx.eps, *need)
        else:
            dx, dw, db = norm_backward(dy, x, weight, ctx.groups, ctx.eps, *need)
        return (dx if need[0] else None, dw.view(ctx.table[0]).to(ctx.table[1]) if need[1] else None,
                db.view(ctx.bias[0]).to(ctx.bias[1]) if need[2] else None, None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of the last dimension; weight and bias [D], or [G, D] over the last two dimensions, or None."""
    eps = float(eps)
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
        if weight is not None and bias is not None and weight.shape != bias.shape:
            raise ValueError(f"weight {tuple(weight.shape)} and bias {tuple(bias.shape)} must share a shape")
        if t.ndim == 2:
            groups = t.shape[0]
    if groups < 1:
        raise ValueError("weight and bias need at least one group")
    _launch.check_dtype("x", x)
    _launch.check_device(x, weight=weight, bias=bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFn.apply(x, weight, bias, groups, eps)
    if torch.compiler.is_compiling():
        return torch.ops.dwarf.layer_norm_fwd(x, weight, bias, groups, eps)
    return norm_forward(x, weight, bias, groups, eps)
