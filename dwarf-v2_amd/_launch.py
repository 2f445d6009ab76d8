"""Host-side pieces of the mixers' operators (norm.py, rotary.py, linattn.py, conv.py, selscan.py): the native module, and
the argument checks of compiled and traced calls."""

from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.DWARF_BF16, torch.float16: _lib.DWARF_F16, torch.float32: _lib.DWARF_F32}
_NATIVE = None


def native():
    """The module ``_mixer`` (csrc/mixer_torch.cpp, csrc/selective_torch.cpp): checks, buffers, autograd nodes and launches of eager calls."""
    global _NATIVE
    if _NATIVE is None:
        _lib.load()   # its ABI is checked first
        try:
            from . import _mixer
        except ImportError as e:
            raise _lib.NativeLibraryError(f"_mixer.so is not built for this Python and torch ({e}); build it with "
                                          "`make -C dwarf-v2_amd/csrc` or __graft_entry__.build()") from e
        if _mixer.abi_version != _lib.ABI_VERSION:
            raise _lib.NativeLibraryError(f"_mixer.so ABI {_mixer.abi_version} does not match the binding's ABI "
                                          f"{_lib.ABI_VERSION}")
        _mixer.set_error_class(_lib.NativeLibraryError)
        _NATIVE = _mixer
    return _NATIVE


def check_dtype(what: str, x: torch.Tensor) -> None:
    if x.dtype not in DTYPES:
        raise ValueError(f"{what} must be bf16, fp16 or fp32, got {x.dtype}")


def check_device(x: torch.Tensor, **others) -> None:
    """Device tensors, all on one device."""
    if not x.is_cuda:
        raise RuntimeError("the mixer's HIP kernels require device tensors")
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, expected {x.device}")


def check_channels(name: str, t: torch.Tensor | None, D: int) -> None:
    """A table of one floating value for each channel."""
    if t is not None and (tuple(t.shape) != (D,) or not t.is_floating_point()):
        raise ValueError(f"{name} must be [{D}] floating point, got {tuple(t.shape)} {t.dtype}")


def check_lengths(lengths: torch.Tensor | None, B: int) -> None:
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"lengths must be [{B}] int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")


def check_slots(slots: torch.Tensor | None, rows: int) -> None:
    if slots is not None and (tuple(slots.shape) != (rows,) or slots.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"slots must be [{rows}] int32 or int64, got {tuple(slots.shape)} {slots.dtype}")


def check_pools(state: torch.Tensor, new_state: torch.Tensor | None, slots: torch.Tensor | None, rows: int,
                each: tuple[int, int], dtype: torch.dtype) -> None:
    """A pool [P, *each] of states, and the one that the new ones go to."""
    for name, t in (("state", state), ("new_state", new_state)):
        if t is not None and (t.dtype != dtype or t.ndim != 3 or tuple(t.shape[1:]) != each):
            raise ValueError(f"{name} must be a {dtype} [P,{each[0]},{each[1]}] pool, got {tuple(t.shape)} {t.dtype}")
    if new_state is not None and new_state.shape != state.shape:
        raise ValueError("new_state must have state's shape and strides")
    if slots is None and state.shape[0] < rows:
        raise ValueError(f"a pool of {state.shape[0]} states does not hold the {rows} rows")
