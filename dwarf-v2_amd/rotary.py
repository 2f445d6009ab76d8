"""Rotary positions of q and k on MI355X, in one launch, with their gradients.

``rotary_plan`` holds the angle per position of each pair of elements, for one
device, and how the pairs lie: side by side (``interleaved=True``) or half a
rotary width apart.  ``rotary_embed(q, k, positions, plan)`` turns the first
``rotary_dim`` elements of every row and copies the rest.

The angles are held as 64-bit fractions of a turn, so that position times
angle wraps exactly: positions of 2^31 are as exact as small ones, where a
product in fp32 is off by 0.03 rad at position 2^20.
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch
from torch.autograd.function import once_differentiable

from . import _launch

_TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
SCALINGS = (None, "linear", "base", "bands")


class RotaryPlan:
    """Angles per position on one device: ``turns`` [pairs] int64 (2^-64 turns), ``inverse_frequencies`` [pairs]
    float64 on the CPU, ``rotary_dim``, ``interleaved``, ``magnitude``."""

    def __init__(self, inverse_frequencies: torch.Tensor, interleaved: bool, magnitude: float, device):
        f = inverse_frequencies.detach().to(device="cpu", dtype=torch.float64).reshape(-1)
        if f.numel() < 1 or not bool(torch.isfinite(f).all()):
            raise ValueError("inverse_frequencies must be finite, one for each pair")
        if not math.isfinite(float(magnitude)):
            raise ValueError("magnitude must be finite")
        turns = [int(Fraction(x) / _TWO_PI * 2 ** 64 + Fraction(1, 2)) % 2 ** 64 for x in f.tolist()]
        self.inverse_frequencies = f
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
        self.rotary_dim, self.interleaved, self.magnitude = 2 * f.numel(), bool(interleaved), float(magnitude)

    def to(self, device) -> "RotaryPlan":
        """The same plan on another device."""
        return RotaryPlan(self.inverse_frequencies, self.interleaved, self.magnitude, device)


def rotary_plan(rotary_dim: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str | None = None,
                factor: float = 1.0, original_length: int | None = None, fast_turns: float = 32.0,
                slow_turns: float = 1.0, magnitude: float = 1.0, inverse_frequencies: torch.Tensor | None = None,
                device=None) -> RotaryPlan:
    """The plan of pairs i at base^(-2i / rotary_dim) radians per position, or at ``inverse_frequencies``
    [rotary_dim / 2].  scaling stretches them for contexts ``factor`` times as long:

    "linear"  every frequency over ``factor`` (positions are compressed);
    "base"    a base factor^(d / (d - 2)) times as large: the fastest pair stays, the slowest is stretched;
    "bands"   by the turns a pair makes over ``original_length`` positions: ``fast_turns`` or more keep their
              frequency, ``slow_turns`` or fewer are divided by ``factor``, a linear mixture between.

    magnitude scales the turned elements."""
    rotary_dim = int(rotary_dim)
    base, factor = float(base), float(factor)
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError("base and factor must be finite and positive")
    if scaling == "base":
        if rotary_dim < 4 or inverse_frequencies is not None:
            raise ValueError("scaling='base' needs rotary_dim of at least 4 and no inverse_frequencies of its own")
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    if inverse_frequencies is None:
        f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    else:
        f = inverse_frequencies.detach().to(device="cpu", dtype=torch.float64).reshape(-1)
        if f.numel() != rotary_dim // 2:
            raise ValueError(f"inverse_frequencies must hold {rotary_dim // 2} values, got {f.numel()}")
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        if original_length is None or int(original_length) < 1:
            raise ValueError("scaling='bands' needs original_length")
        if not (math.isfinite(fast_turns) and math.isfinite(slow_turns) and fast_turns > slow_turns):
            raise ValueError("fast_turns must be above slow_turns")
        turns = int(original_length) * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / factor
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return RotaryPlan(f, interleaved, magnitude, device)


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, turns: torch.Tensor, interleaved: bool,
           inverse: bool, magnitude: float) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Raw launch: the turned (q, k), in token-major memory."""
    return _launch.native().rotate(q, k, positions, turns, interleaved, inverse, magnitude)


class _RotaryFn(torch.autograd.Function):
    """The autograd node of compiled and traced calls; eager calls have theirs in C++."""

    @staticmethod
    def forward(ctx, q, k, positions, turns, interleaved: bool, magnitude: float):
        ctx.save_for_backward(positions, turns)
        ctx.how = (interleaved, magnitude, k is not None)
        q_out, k_out = torch.ops.dwarf.rotary(q, k, positions, turns, interleaved, False, magnitude)
        return (q_out, k_out) if k is not None else (q_out, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, turns = ctx.saved_tensors
        interleaved, magnitude, has_k = ctx.how
        gq, gk = torch.ops.dwarf.rotary(dq, dk if has_k else None, positions, turns, interleaved, True, magnitude)
        return gq, gk if has_k else None, None, None, None, None


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 plan: RotaryPlan) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q [B,H,N,D] and k [B,H_kv,N,D] (or None) turned to their positions, [N] or [B,N] int32 or int64.

    bf16, fp16 or fp32, any strides with a unit last one; D even, at least the plan's rotary_dim.  The results
    have q's and k's shapes in [B,N,H,D] memory."""
    if not torch.compiler.is_compiling():
        turned = _launch.native().rotary_embed(q, k, positions, plan.turns, plan.interleaved, plan.magnitude)
        if turned is not None:   # None: fake or wrapped tensors, a mode or a trace
            return turned
    _check(q, k, positions, plan)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RotaryFn.apply(q, k, positions, plan.turns, plan.interleaved, plan.magnitude)
    q_out, k_out = torch.ops.dwarf.rotary(q, k, positions, plan.turns, plan.interleaved, False, plan.magnitude)
    return q_out, (k_out if k is not None else None)


def _check(q, k, positions, plan) -> None:
    """The native call's checks, for compiled and traced calls."""
    if q.ndim != 4:
        raise ValueError(f"q must be [B,H,N,D], got {tuple(q.shape)}")
    B, H, N, D = q.shape
    if k is not None and (k.ndim != 4 or (k.shape[0], k.shape[2], k.shape[3]) != (B, N, D) or k.dtype != q.dtype):
        raise ValueError(f"k must be [B,H_kv,N,D] like q {tuple(q.shape)} {q.dtype}, got {tuple(k.shape)} {k.dtype}")
    if D % 2 or plan.rotary_dim > D:
        raise ValueError(f"D={D} must be even and at least the plan's rotary_dim {plan.rotary_dim}")
    if H < 1 or (k is not None and k.shape[1] < 1):
        raise ValueError("q and k need at least one head")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if tuple(positions.shape) not in ((N,), (B, N)):
        raise ValueError(f"positions must be [{N}] or [{B},{N}], got {tuple(positions.shape)}")
    _launch.check_dtype("q", q)
    _launch.check_device(q, k=k, positions=positions, plan=plan.turns)
