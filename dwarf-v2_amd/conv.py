"""A short causal convolution of each channel on MI355X: prompts, training and single tokens.

    p_t = bias + sum_j weight[:, j] x_{t-W+1+j},    y_t = p_t or silu(p_t)

``causal_conv`` runs whole sequences (with gradients for x, weight, bias and the
state that enters); ``causal_conv_step`` runs one token of each running sequence
against a pool of states.  A sequence's state is its last W - 1 inputs.  Rows are
bf16, fp16 or fp32, sums fp32 and rounded once; weight and bias may have any
floating dtype (used in fp32, their gradients are summed in a fixed order).
W is 1 to 8.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _launch

MAX_WIDTH = 8


def conv_forward(x, weight, bias, initial, lengths, silu: bool, want_state: bool
                 ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Raw launch: (y contiguous, the final state or None)."""
    return _launch.native().conv_forward(x, weight, bias, initial, lengths, silu, want_state)


def conv_backward(dy, dstate, x, weight, bias, initial, lengths, silu: bool, need_w: bool, need_b: bool,
                  need_initial: bool):
    """Raw launches: (dx, dweight and dbias fp32, dinitial); None where not needed."""
    return _launch.native().conv_backward(dy, dstate, x, weight, bias, initial, lengths, silu, need_w, need_b,
                                          need_initial)


def conv_step(x, weight, bias, state, new_state, slots, silu: bool) -> torch.Tensor:
    """Raw launch of one step: out [rows, D]; new_state None writes the pool itself."""
    return _launch.native().conv_step(x, weight, bias, state, new_state, slots, silu)


class _CausalConvFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, silu: bool, want_state: bool):
        ctx.set_materialize_grads(False)
        y, state = torch.ops.dwarf.causal_conv_fwd(x, weight, bias, initial, lengths, silu, want_state)
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and dstate is None:
            return (None,) * 7
        if dy is None:
            dy = torch.zeros_like(x)
        dx, dw, db, di = torch.ops.dwarf.causal_conv_bwd(dy, dstate, x, weight, bias, initial, lengths, ctx.silu, need[1],
                                                         need[2], need[3])
        return (dx, dw.to(weight.dtype) if need[1] else None, db.to(bias.dtype) if need[2] else None,
                di if need[3] else None, None, None, None)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                activation: str | None = None, initial_state: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None, return_state: bool = False):
    """Causal convolution of each channel over whole sequences: y [B,N,D] in x's dtype, and with ``return_state`` the
    state [B,W-1,D] behind each sequence's last token.

    x [B,N,D]; weight [D,W], its last tap on the token itself; bias [D]; activation None or "silu"; initial_state
    [B,W-1,D] in x's dtype, the inputs in front of the first token (zeros without it); lengths [B] integers, clamped to
    [0, N]: the tokens of each sequence, behind which nothing is used and the output is zero."""
    silu = _check_activation(activation)
    if not torch.compiler.is_compiling():
        done = _launch.native().causal_conv(x, weight, bias, silu, initial_state, lengths, return_state)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    _check(x, weight, bias, initial_state, lengths)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, initial_state)):
        return _CausalConvFn.apply(x, weight, bias, initial_state, lengths, silu, bool(return_state))
    y, state = torch.ops.dwarf.causal_conv_fwd(x, weight, bias, initial_state, lengths, silu, bool(return_state))
    return (y, state) if return_state else y


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, state: torch.Tensor, *,
                     activation: str | None = None, slots: torch.Tensor | None = None,
                     new_state: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each row: x [rows,D]; returns out [rows,D].

    state [P,W-1,D] in x's dtype is a pool of sequences' last inputs, each slot contiguous.  Row r works on slot slots[r]
    (slot r where slots is None); its inputs moved on by one are written to the same slot of ``new_state``, or of
    ``state`` itself where that is None.  Slots outside [0, P) mark rows that pad the batch: no state is touched, their
    output is zero.  Rows that share a slot are consecutive tokens of its sequence, in row order.  No gradients."""
    silu = _check_activation(activation)
    if not torch.compiler.is_compiling():
        done = _launch.native().causal_conv_step(x, weight, bias, state, silu, slots, new_state)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    _check_step(x, weight, bias, state, slots, new_state)
    if new_state is None:
        return torch.ops.dwarf.causal_conv_step_(x, weight, bias, state, slots, silu)
    return torch.ops.dwarf.causal_conv_step(x, weight, bias, state, new_state, slots, silu)


def _check_activation(activation) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f'activation must be None or "silu", got {activation!r}')
    return activation == "silu"


def _check_taps(weight, bias, D: int) -> None:
    if weight.ndim != 2 or weight.shape[0] != D or weight.shape[1] < 1 or not weight.is_floating_point():
        raise ValueError(f"weight must be [{D},W] floating point, got {tuple(weight.shape)} {weight.dtype}")
    if weight.shape[1] > MAX_WIDTH:
        raise RuntimeError(f"the convolution is built for W up to {MAX_WIDTH}, got {weight.shape[1]}")
    _launch.check_channels("bias", bias, D)


def _check(x, weight, bias, initial_state, lengths) -> None:
    """The native call's checks, for compiled and traced calls."""
    if x.ndim != 3 or x.shape[2] < 1:
        raise ValueError(f"x must be [B,N,D], got {tuple(x.shape)}")
    _launch.check_dtype("x", x)
    B, _, D = x.shape
    _check_taps(weight, bias, D)
    shape = (B, weight.shape[1] - 1, D)
    if initial_state is not None and (tuple(initial_state.shape) != shape or initial_state.dtype != x.dtype):
        raise ValueError(f"initial_state must be {x.dtype} {list(shape)}, got {tuple(initial_state.shape)} "
                         f"{initial_state.dtype}")
    _launch.check_lengths(lengths, B)
    _launch.check_device(x, weight=weight, bias=bias, initial_state=initial_state, lengths=lengths)


def _check_step(x, weight, bias, state, slots, new_state) -> None:
    """The native call's checks but those of memory (strides and overlaps, made at the launch), for compiled and traced
    calls."""
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows,D], got {tuple(x.shape)}")
    _launch.check_dtype("x", x)
    R, D = x.shape
    _check_taps(weight, bias, D)
    _launch.check_slots(slots, R)
    _launch.check_pools(state, new_state, slots, R, (weight.shape[1] - 1, D), x.dtype)
    _launch.check_device(x, weight=weight, bias=bias, state=state, new_state=new_state, slots=slots)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state, new_state)):
        raise RuntimeError("causal_conv_step has no gradients: call it under torch.no_grad(), or causal_conv")
