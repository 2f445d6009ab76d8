"""Host-side pieces of the mixer's operators (norm.py, rotary.py, linattn.py): the native module, and the argument
checks of compiled and traced calls."""

from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.DWARF_BF16, torch.float16: _lib.DWARF_F16, torch.float32: _lib.DWARF_F32}
_NATIVE = None


def native():
    """The module ``_mixer`` (csrc/mixer_torch.cpp): checks, buffers, autograd nodes and launches of eager calls."""
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
