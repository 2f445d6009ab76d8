"""Host-side pieces of the mixer's operators (norm.py, rotary.py, linattn.py): element types and launches."""

from __future__ import annotations

import ctypes

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.DWARF_BF16, torch.float16: _lib.DWARF_F16, torch.float32: _lib.DWARF_F32}


def launch(name: str, args, device: torch.device) -> None:
    """Calls the entry point on the device's current stream, with the device current for the launch."""
    fn = getattr(_lib.load(), name)
    if device.index is not None and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream)
    if rc:
        _lib.check(rc, name)


def workspace(name: str, args, device: torch.device) -> torch.Tensor | None:
    """The bytes that an entry point's ``*_bytes`` call asks for (None: none)."""
    nbytes = int(getattr(_lib.load(), name)(ctypes.byref(args)))
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def check_dtype(what: str, x: torch.Tensor) -> int:
    if x.dtype not in DTYPES:
        raise ValueError(f"{what} must be bf16, fp16 or fp32, got {x.dtype}")
    return DTYPES[x.dtype]


def check_device(x: torch.Tensor, **others) -> None:
    """Device tensors, all on one device."""
    if not x.is_cuda:
        raise RuntimeError("the mixer's HIP kernels require device tensors")
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, expected {x.device}")


def token_major(B: int, H: int, N: int, D: int, like: torch.Tensor) -> torch.Tensor:
    """An empty [B,H,N,D] tensor in [B,N,H,D] memory: ``transpose(1, 2).reshape(B, N, H * D)`` is a view."""
    return torch.empty((B, N, H, D), device=like.device, dtype=like.dtype).transpose(1, 2)
