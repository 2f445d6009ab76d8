"""The selective scan on MI355X: prompts, training and single tokens.

For each channel, with its S states,

    step = delta + delta_bias (through a softplus, where asked),  a = exp(step A)
    h_t = a h_{t-1} + step x_t B_t,    y_t = (C_t . h_t + skip x_t) silu(gate_t)

``causal_ema_scan``'s recurrence with a rate, an input weight and an output
weight that each token chooses.  ``selective_scan`` runs whole sequences (with
gradients for every input and the state that enters); ``selective_scan_step``
runs one token of each running sequence against a pool of states.  States and
sums are fp32; x, delta, gate, B and C are bf16, fp16 or fp32; S is 1 to 64, and
groups of channels may share their B and C.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _launch

MAX_STATES = 64


def checkpoint_elements(B: int, N: int, D: int, S: int) -> int:
    """fp32 elements that the forward keeps for the backward (dwarf_selective_scan_checkpoint_bytes): the padded states in
    front of each chunk."""
    per_lane = 2 if S <= 8 else 4 if S <= 16 else 8
    chunk = 64 // per_lane
    return B * -(-N // chunk) * D * per_lane * (4 if S <= 32 else 8)


def scan_forward(x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, softplus: bool, want_state: bool,
                 want_checkpoints: bool) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """Raw launches: (y contiguous, the final state or None, the backward's checkpoints or None)."""
    return _launch.native().scan_forward(x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, softplus, want_state,
                                         want_checkpoints)


def scan_backward(dy, dstate, x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, checkpoints, softplus: bool,
                  need_A: bool, need_skip: bool, need_bias: bool, need_initial: bool):
    """Raw launches: (dx, ddelta, dA, dB, dC, dskip, dgate, ddelta_bias, dinitial); dA, dskip, ddelta_bias and dinitial
    fp32, None where not needed."""
    return _launch.native().scan_backward(dy, dstate, x, delta, A, B, C, skip, gate, delta_bias, initial, lengths,
                                          checkpoints, softplus, need_A, need_skip, need_bias, need_initial)


def scan_step(x, delta, A, B, C, state, new_state, skip, gate, delta_bias, slots, softplus: bool) -> torch.Tensor:
    """Raw launch of one step: out [rows, D]; new_state None writes the pool itself."""
    return _launch.native().scan_step(x, delta, A, B, C, state, new_state, skip, gate, delta_bias, slots, softplus)


class _SelectiveScanFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, softplus: bool, want_state: bool):
        ctx.set_materialize_grads(False)
        y, state, checkpoints = torch.ops.dwarf.selective_scan_fwd(x, delta, A, B, C, skip, gate, delta_bias, initial,
                                                                   lengths, softplus, want_state, True)
        ctx.save_for_backward(x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, checkpoints)
        ctx.softplus = softplus
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, checkpoints = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None and dstate is None:
            return (None,) * 12
        if dy is None:
            dy = torch.zeros_like(x)
        dx, dd, dA, dB, dC, dskip, dgate, dbias, dinitial = torch.ops.dwarf.selective_scan_bwd(
            dy, dstate, x, delta, A, B, C, skip, gate, delta_bias, initial, lengths, checkpoints, ctx.softplus, need[2],
            need[5], need[7], need[8])
        return (dx, dd, dA.to(A.dtype) if need[2] else None, dB, dC, dskip.to(skip.dtype) if need[5] else None,
                dgate if need[6] else None, dbias.to(delta_bias.dtype) if need[7] else None,
                dinitial if need[8] else None, None, None, None)


def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   skip: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                   delta_bias: torch.Tensor | None = None, softplus: bool = False,
                   initial_state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   return_state: bool = False):
    """Selective scan over whole sequences: y [B,N,D] in x's dtype, and with ``return_state`` the state [B,D,S] fp32 behind
    each sequence's last token.

    x, delta and gate [B,N,D]; A [D,S], below 0 for states that decay; B and C [B,N,S], or [B,N,G,S] for G groups of D/G
    adjacent channels; skip and delta_bias [D]; A, skip and delta_bias of any floating dtype; initial_state [B,D,S] fp32;
    lengths [B] integers, clamped to [0, N]: the tokens of each sequence, behind which nothing is used and the output is
    zero."""
    if not torch.compiler.is_compiling():
        done = _launch.native().selective_scan(x, delta, A, B, C, skip, gate, delta_bias, softplus, initial_state, lengths,
                                               return_state)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    _check(x, delta, A, B, C, skip, gate, delta_bias, initial_state, lengths)
    given = (x, delta, A, B, C, skip, gate, delta_bias, initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        return _SelectiveScanFn.apply(*given, lengths, bool(softplus), bool(return_state))
    y, state, _ = torch.ops.dwarf.selective_scan_fwd(*given, lengths, bool(softplus), bool(return_state), False)
    return (y, state) if return_state else y


def selective_scan_step(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, *, skip: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                        delta_bias: torch.Tensor | None = None, softplus: bool = False,
                        slots: torch.Tensor | None = None, new_state: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each row: x, delta and gate [rows,D], B and C [rows,S] or [rows,G,S]; returns out [rows,D].

    state [P,D,S] fp32 is a pool of sequences' states, each slot contiguous.  Row r works on slot slots[r] (slot r where
    slots is None); its new state is written to the same slot of ``new_state``, or of ``state`` itself where that is
    None.  Slots outside [0, P) mark rows that pad the batch: no state is touched, their output is zero.  Rows that share
    a slot are consecutive tokens of its sequence, in row order.  No gradients."""
    if not torch.compiler.is_compiling():
        done = _launch.native().selective_scan_step(x, delta, A, B, C, state, skip, gate, delta_bias, softplus, slots,
                                                    new_state)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    _check_step(x, delta, A, B, C, state, skip, gate, delta_bias, slots, new_state)
    if new_state is None:
        return torch.ops.dwarf.selective_scan_step_(x, delta, A, B, C, state, skip, gate, delta_bias, slots, bool(softplus))
    return torch.ops.dwarf.selective_scan_step(x, delta, A, B, C, state, new_state, skip, gate, delta_bias, slots,
                                               bool(softplus))


def _check_inputs(x, delta, A, B, C, skip, gate, delta_bias, dims: str) -> None:
    D, lead = x.shape[-1], x.ndim - 1
    _launch.check_dtype("x", x)
    for name, t in (("delta", delta), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{name} must be {tuple(x.shape)} {x.dtype} as x is, got {tuple(t.shape)} {t.dtype}")
    if A.ndim != 2 or A.shape[0] != D or A.shape[1] < 1 or not A.is_floating_point():
        raise ValueError(f"A must be [{D},S] floating point, got {tuple(A.shape)} {A.dtype}")
    S = A.shape[1]
    for name, t in (("B", B), ("C", C)):
        if (t.ndim not in (lead + 1, lead + 2) or t.shape[:lead] != x.shape[:lead] or t.shape[-1] != S
                or t.dtype != x.dtype):
            raise ValueError(f"{name} must be {x.dtype} [{dims},G,{S}] or [{dims},{S}] for x {tuple(x.shape)}, got "
                             f"{tuple(t.shape)} {t.dtype}")
    if B.shape != C.shape:
        raise ValueError(f"B and C must share a shape, got {tuple(B.shape)} and {tuple(C.shape)}")
    G = B.shape[-2] if B.ndim == lead + 2 else 1
    if G < 1 or D % G:
        raise ValueError(f"D={D} channels must be divisible by G={G} groups")
    if S > MAX_STATES:
        raise RuntimeError(f"the scan is built for up to {MAX_STATES} states, got {S}")
    _launch.check_channels("skip", skip, D)
    _launch.check_channels("delta_bias", delta_bias, D)
    _launch.check_device(x, delta=delta, A=A, B=B, C=C, skip=skip, gate=gate, delta_bias=delta_bias)


def _check(x, delta, A, B, C, skip, gate, delta_bias, initial_state, lengths) -> None:
    """The native call's checks, for compiled and traced calls."""
    if x.ndim != 3 or x.shape[2] < 1:
        raise ValueError(f"x must be [B,N,D], got {tuple(x.shape)}")
    _check_inputs(x, delta, A, B, C, skip, gate, delta_bias, "B,N")
    shape = (x.shape[0], x.shape[2], A.shape[1])
    if initial_state is not None and (tuple(initial_state.shape) != shape or initial_state.dtype != torch.float32):
        raise ValueError(f"initial_state must be fp32 {list(shape)}, got {tuple(initial_state.shape)} {initial_state.dtype}")
    _launch.check_lengths(lengths, x.shape[0])
    _launch.check_device(x, initial_state=initial_state, lengths=lengths)


def _check_step(x, delta, A, B, C, state, skip, gate, delta_bias, slots, new_state) -> None:
    """The native call's checks but those of memory (strides and overlaps, made at the launch), for compiled and traced
    calls."""
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows,D], got {tuple(x.shape)}")
    _check_inputs(x, delta, A, B, C, skip, gate, delta_bias, "rows")
    _launch.check_slots(slots, x.shape[0])
    _launch.check_pools(state, new_state, slots, x.shape[0], (x.shape[1], A.shape[1]), torch.float32)
    _launch.check_device(x, state=state, new_state=new_state, slots=slots)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, delta, A, B, C, state, skip, gate,
                                                                                   delta_bias, new_state)):
        raise RuntimeError("selective_scan_step has no gradients: call it under torch.no_grad(), or selective_scan")
