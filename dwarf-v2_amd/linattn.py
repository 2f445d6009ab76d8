"""Linear attention with a decay for each head, on MI355X: prompts, training and single tokens.

With g = exp(log_decay[h]) <= 1 a head keeps one 64 x 64 state,

    S_t = g S_{t-1} + k_t v_t^T,    o_t = scale q_t S_t,

the matrix form of ``causal_ema_scan``'s recurrence, whose serving state does
not grow with the context.  ``linear_attention`` runs whole sequences in chunks
on the matrix cores (with gradients for q, k, v, log_decay and the state that
enters); ``linear_attention_step`` runs one token of each running sequence
against a pool of states.  States and sums are fp32; q, k, v are bf16, fp16 or
fp32; head_dim is 64, the query heads a multiple of the K/V heads.
"""

from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _launch
from .dsqg import HEAD_DIM


def segment_tokens(B: int, H: int, N: int) -> int:
    """Tokens of a segment (dwarf_linear_attention_segment): shorter ones where long ones leave CUs idle."""
    for seg in (1024, 512, 256, 128):
        if B * H * -(-N // seg) >= (448 if seg >= 512 else 224):
            return seg
    return 64


def states_shape(B: int, H: int, N: int) -> tuple[int, ...]:
    """Shape of the states the forward keeps for the backward: one per segment, none for a single segment."""
    segs = -(-N // segment_tokens(B, H, N)) if B * H * N else 0
    return (B, H, segs if segs > 1 else 0, HEAD_DIM, HEAD_DIM)


def attention_forward(q, k, v, log_decay, initial, lengths, scale: float, want_state: bool
                      ) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """Raw launches: (out in token-major memory, the final state or None, the segments' states)."""
    return _launch.native().attention_forward(q, k, v, log_decay, initial, lengths, scale, want_state)


def attention_backward(dout, dstate, q, k, v, log_decay, initial, lengths, scale: float, states, state,
                       need_decay: bool, need_initial: bool):
    """Raw launches: (dq, dk, dv in token-major memory, dlog_decay [H] or None, dinitial or None)."""
    return _launch.native().attention_backward(dout, dstate, q, k, v, log_decay, initial, lengths, scale, states, state,
                                               need_decay, need_initial)


def attention_step(q, k, v, log_decay, state, new_state, slots, scale: float, out=None) -> torch.Tensor:
    """Raw launch of one step: out [S,H,64]; new_state None writes the pool itself."""
    return _launch.native().attention_step(q, k, v, log_decay, state, new_state, slots, scale, out)


class _LinearAttentionFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale: float, want_state: bool):
        out, state, states = torch.ops.dwarf.linear_attention_fwd(q, k, v, log_decay, initial, lengths, scale, want_state)
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths, states, state if want_state else None)
        ctx.scale = scale
        return (out, state) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstate=None):
        q, k, v, log_decay, initial, lengths, states, state = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dlog, dinitial = torch.ops.dwarf.linear_attention_bwd(
            dout, dstate, q, k, v, log_decay, initial, lengths, ctx.scale, states, state, need[3], need[4])
        return (dq, dk, dv, dlog.view(log_decay.shape).to(log_decay.dtype) if need[3] else None,
                dinitial if need[4] else None, None, None, None)


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     scale: float | None = None, initial_state: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, return_state: bool = False):
    """Decayed linear attention over whole sequences: out [B,H,N,64] in q's dtype ([B,N,H,64] memory), and with
    ``return_state`` the state [B,H,64,64] fp32 behind each sequence's last token.

    q [B,H,N,64], k and v [B,H_kv,N,64]; log_decay [H], values above 0 count as 0 (their gradient is 0);
    scale 1/8 by default; initial_state [B,H,64,64] fp32; lengths [B] integers, clamped to [0, N]: the tokens of
    each sequence, behind which nothing is used and the output is zero.  Tokens are summed 64 at a time, so one
    that is not finite spoils its sequence's outputs from the first of its 64 on."""
    if not torch.compiler.is_compiling():
        done = _launch.native().linear_attention(q, k, v, log_decay, scale, initial_state, lengths, return_state)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    scale = _check(q, k, v, log_decay, scale, initial_state, lengths)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        return _LinearAttentionFn.apply(q, k, v, log_decay, initial_state, lengths, scale, bool(return_state))
    out, state, _ = torch.ops.dwarf.linear_attention_fwd(q, k, v, log_decay, initial_state, lengths, scale, bool(return_state))
    return (out, state) if return_state else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, slots: torch.Tensor | None = None,
                          new_state: torch.Tensor | None = None, scale: float | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of each of S rows: q [S,H,64], k and v [S,H_kv,64]; returns out [S,H,64].

    state [P,H,64,64] fp32 is a pool of sequences' states, each slot contiguous.  Row s works on slot slots[s]
    (slot s where slots is None); its new state is written to the same slot of ``new_state``, or of ``state`` itself
    where that is None.  Slots outside [0, P) mark rows that pad the batch: no state is touched, their output
    is zero.  Rows that share a slot are consecutive tokens of its sequence, in row order.  ``out``: where to write
    the result (eager calls), in memory of its own: it may lie between the rows of the others, but not on them.  No
    gradients."""
    if not torch.compiler.is_compiling():
        done = _launch.native().linear_attention_step(q, k, v, log_decay, state, slots, new_state, scale, out)
        if done is not None:   # None: fake or wrapped tensors, a mode or a trace
            return done
    elif out is not None:
        raise RuntimeError("out= is for eager calls and captured graphs, not for torch.compile")
    scale = _check_step(q, k, v, log_decay, state, slots, new_state, scale, out)
    if new_state is None:
        result = torch.ops.dwarf.linear_attention_step_(q, k, v, log_decay, state, slots, scale)
    else:
        result = torch.ops.dwarf.linear_attention_step(q, k, v, log_decay, state, new_state, slots, scale)
    return result if out is None else out.copy_(result)


def _check_scale(scale) -> float:
    scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return scale


def _check_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, dims: str) -> None:
    H, Hkv = q.shape[1], k.shape[1]
    if k.shape != v.shape or q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"k and v must share a shape and q's dtype {q.dtype}; got {tuple(k.shape)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)} ({dims})")
    if Hkv < 1 or H < 1 or H % Hkv:
        raise ValueError(f"num query heads H={H} must be divisible by KV heads H_kv={Hkv}")
    if log_decay.numel() != H or not log_decay.is_floating_point():
        raise ValueError(f"log_decay must hold one floating value per head ({H}), got {tuple(log_decay.shape)} {log_decay.dtype}")
    _launch.check_dtype("q", q)


def _check(q, k, v, log_decay, scale, initial_state, lengths) -> float:
    """The native call's checks, for compiled and traced calls; returns the scale."""
    scale = _check_scale(scale)
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError(f"q, k and v must be [B,H,N,{HEAD_DIM}], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    _check_heads(q, k, v, log_decay, "[B,H,N,64]")
    B, H, N, hd = q.shape
    if initial_state is not None and (tuple(initial_state.shape) != (B, H, hd, hd) or initial_state.dtype != torch.float32):
        raise ValueError(f"initial_state must be fp32 [{B},{H},{hd},{hd}], got {tuple(initial_state.shape)} "
                         f"{initial_state.dtype}")
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"lengths must be [{B}] int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")
    _launch.check_device(q, k=k, v=v, log_decay=log_decay, initial_state=initial_state, lengths=lengths)
    if hd != HEAD_DIM:
        raise RuntimeError(f"linear attention is built for head_dim {HEAD_DIM}, got {hd}")
    return scale


def _check_step(q, k, v, log_decay, state, slots, new_state, scale, out) -> float:
    """The native call's checks but those of memory (strides and alignment, made at the launch), for compiled and traced
    calls."""
    scale = _check_scale(scale)
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError(f"q, k and v must be [S,H,{HEAD_DIM}], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    _check_heads(q, k, v, log_decay, "[S,H,64]")
    S, H, hd = q.shape
    if hd != HEAD_DIM:
        raise RuntimeError(f"linear attention is built for head_dim {HEAD_DIM}, got {hd}")
    for name, t in (("state", state), ("new_state", new_state)):
        if t is not None and (t.dtype != torch.float32 or t.ndim != 4 or tuple(t.shape[1:]) != (H, hd, hd)):
            raise ValueError(f"{name} must be an fp32 [P,{H},{hd},{hd}] pool, got {tuple(t.shape)} {t.dtype}")
    if new_state is not None and new_state.shape != state.shape:
        raise ValueError("new_state must have state's shape and strides")
    if slots is None and state.shape[0] < S:
        raise ValueError(f"a pool of {state.shape[0]} states does not hold the {S} rows")
    if slots is not None and (tuple(slots.shape) != (S,) or slots.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"slots must be [{S}] int32 or int64, got {tuple(slots.shape)} {slots.dtype}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype}, got {tuple(out.shape)} {out.dtype}")
    _launch.check_device(q, k=k, v=v, log_decay=log_decay, state=state, new_state=new_state, slots=slots, out=out)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (q, k, v, log_decay, state, new_state, out)):
        raise RuntimeError("linear_attention_step has no gradients: call it under torch.no_grad(), or linear_attention")
    return scale
