"""Host side of the selective mixer's operators, without a GPU: the header's exports and layouts, refusals of bad calls,
sizes that both sides of the C ABI compute, fake shapes."""

import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from tests.conftest import ROOT

HEADER = os.path.join(ROOT, "include", "dwarf_selective.h")
STRUCTS = {"dwarf_rms_norm_fwd_args": "RmsNormFwdArgs", "dwarf_rms_norm_bwd_args": "RmsNormBwdArgs",
           "dwarf_causal_conv_fwd_args": "CausalConvFwdArgs", "dwarf_causal_conv_bwd_args": "CausalConvBwdArgs",
           "dwarf_causal_conv_step_args": "CausalConvStepArgs", "dwarf_selective_scan_fwd_args": "SelectiveScanFwdArgs",
           "dwarf_selective_scan_bwd_args": "SelectiveScanBwdArgs", "dwarf_selective_scan_step_args": "SelectiveScanStepArgs"}
P = 0x10000   # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._lib.load()


def test_header_exports_and_layout(pkg, lib, tmp_path):
    names = sorted(set(re.findall(r"^(?:int|int32_t|size_t)\s+(dwarf_\w+)\s*\(", open(HEADER).read(), re.M)))
    assert sorted(pkg._lib.SELECTIVE_SYMBOLS) == names
    assert all(hasattr(lib, n) for n in names)
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dwarf_selective.h"', "int main(void) {"]
    for cname, pyname in STRUCTS.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in getattr(pkg._lib, pyname)._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, field, value = line.split()
        struct = getattr(pkg._lib, STRUCTS[cname])
        assert (ctypes.sizeof(struct) if field == "sizeof" else getattr(struct, field).offset) == int(value), line


def refused(fn, a, changes, on=None):
    """Each (field, value, status) by itself, then put back."""
    on = a if on is None else on
    for name, value, want in changes:
        keep = getattr(on, name)
        if isinstance(keep, ctypes.Array):
            keep = tuple(keep)
        setattr(on, name, value)
        assert fn(ctypes.byref(a), None) == want, (name, value)
        setattr(on, name, keep)


def test_rms_norm_entry_points_refuse(pkg, lib):
    L = pkg._lib
    bad, no = L.DWARF_ERR_INVALID_ARGUMENT, L.DWARF_ERR_UNSUPPORTED
    assert lib.dwarf_rms_norm_fwd(None, None) == bad and lib.dwarf_rms_norm_bwd(None, None) == bad
    assert lib.dwarf_rms_norm_bwd_workspace_bytes(None) == 0
    f = L.RmsNormFwdArgs()
    f.rows, f.groups, f.D, f.dtype, f.residual_dtype, f.eps = 6, 1, 64, L.DWARF_BF16, L.DWARF_BF16, 1e-5
    f.x = f.y = f.residual = f.sum = P
    f.x_stride = f.y_stride = f.residual_stride = f.sum_stride = (64, 64)
    refused(lib.dwarf_rms_norm_fwd, f, [
        ("x", None, bad), ("x", P + 1, bad), ("y", None, bad), ("y", P + 1, bad), ("residual", P + 1, bad), ("sum", None, bad),
        ("residual_dtype", L.DWARF_F16, bad), ("dtype", 7, bad), ("D", 0, bad), ("groups", 0, bad), ("rows", -1, bad),
        ("eps", -1.0, bad), ("eps", math.nan, bad), ("eps", math.inf, bad), ("groups", 65536, no), ("D", (1 << 24) + 1, no),
        ("rows", 1 << 40, no), ("rows", 0, L.DWARF_OK)])
    f.scale = P
    refused(lib.dwarf_rms_norm_fwd, f, [("y", None, bad)])
    a = L.RmsNormBwdArgs()
    a.rows, a.groups, a.D, a.dtype, a.stream_dtype, a.eps = 6, 1, 64, L.DWARF_BF16, L.DWARF_F32, 1e-5
    a.stream = a.dy = a.dsum = a.dx = a.dresidual = a.dweight = P
    need = lib.dwarf_rms_norm_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    refused(lib.dwarf_rms_norm_bwd, a, [
        ("stream", None, bad), ("stream", P + 2, bad), ("dy", None, bad), ("dsum", P + 2, bad), ("dx", P + 1, bad),
        ("dresidual", P + 2, bad), ("stream_dtype", L.DWARF_F16, bad), ("dtype", 9, bad), ("eps", math.nan, bad), ("D", 0, bad),
        ("rows", -1, bad), ("workspace", None, L.DWARF_ERR_WORKSPACE)])
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.dwarf_rms_norm_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    a.workspace, a.workspace_bytes = P + 4, need
    assert lib.dwarf_rms_norm_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    a.dx = a.dresidual = a.dweight = None
    assert lib.dwarf_rms_norm_bwd(ctypes.byref(a), None) == L.DWARF_OK   # nothing is asked for


def test_causal_conv_entry_points_refuse(pkg, lib):
    L = pkg._lib
    bad, no = L.DWARF_ERR_INVALID_ARGUMENT, L.DWARF_ERR_UNSUPPORTED
    assert all(fn(None, None) == bad for fn in (lib.dwarf_causal_conv_fwd, lib.dwarf_causal_conv_bwd, lib.dwarf_causal_conv_step))
    a = L.CausalConvBwdArgs()
    f = a.fwd
    f.B, f.N, f.D, f.W, f.dtype = 2, 10, 64, 4, L.DWARF_BF16
    f.x = f.y = f.weight = a.dy = a.dx = P
    sizes = [("B", -1, bad), ("N", -1, bad), ("D", 0, bad), ("W", 0, bad), ("W", 9, no), ("dtype", 5, bad), ("N", (1 << 24) + 1, no),
             ("D", (1 << 24) + 1, no), ("weight", None, bad), ("x", None, bad), ("x", P + 1, bad), ("initial", P + 1, bad)]
    refused(lib.dwarf_causal_conv_fwd, f, sizes + [("y", None, bad), ("final", P + 1, bad), ("B", 0, L.DWARF_OK), ("N", 0, L.DWARF_OK)])
    refused(lib.dwarf_causal_conv_bwd, a, sizes, f)
    f.B, f.N, f.D = 1 << 20, 1 << 24, 1 << 10
    assert lib.dwarf_causal_conv_fwd(ctypes.byref(f), None) == no
    f.B, f.N, f.D = 2, 10, 64
    refused(lib.dwarf_causal_conv_bwd, a, [("dy", None, bad), ("dx", None, bad), ("dfinal", P + 1, bad), ("dinitial", P + 1, bad)])
    a.dweight = P
    need = lib.dwarf_causal_conv_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0 and lib.dwarf_causal_conv_bwd_workspace_bytes(None) == 0
    assert lib.dwarf_causal_conv_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.dwarf_causal_conv_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    s = L.CausalConvStepArgs()
    s.R, s.D, s.W, s.pool, s.dtype = 3, 64, 4, 5, L.DWARF_BF16
    s.x = s.out = s.weight = s.state = s.new_state = P
    s.x_stride = s.out_stride = 64
    s.slot_stride = 3 * 64
    refused(lib.dwarf_causal_conv_step, s, [
        ("R", -1, bad), ("D", 0, bad), ("W", 0, bad), ("W", 9, no), ("dtype", 4, bad), ("D", (1 << 24) + 1, no),
        ("R", 1 << 30, no), ("weight", None, bad), ("x", None, bad), ("out", P + 1, bad), ("pool", 2, bad), ("pool", -1, bad),
        ("state", None, bad), ("new_state", None, bad), ("slot_stride", 191, bad), ("new_state", P + 128, bad), ("R", 0, L.DWARF_OK)])
    s.slots, s.pool = P, 0
    assert lib.dwarf_causal_conv_step(ctypes.byref(s), None) == bad   # rows with slots, and none to take


def scan_args(L):
    a = L.SelectiveScanBwdArgs()
    f = a.fwd
    f.B, f.N, f.D, f.G, f.S, f.dtype = 2, 100, 64, 2, 16, L.DWARF_BF16
    f.x = f.delta = f.gate = f.Bm = f.Cm = f.A = f.y = a.dy = a.dx = a.ddelta = a.dgate = a.dB = a.dC = P
    f.x_stride = f.delta_stride = f.gate_stride = f.y_stride = a.dy_stride = a.dx_stride = a.ddelta_stride = a.dgate_stride = (6400, 64)
    f.B_stride = f.C_stride = (3200, 32, 16)
    return a


def test_selective_scan_entry_points_refuse(pkg, lib):
    L = pkg._lib
    bad, no, ws = L.DWARF_ERR_INVALID_ARGUMENT, L.DWARF_ERR_UNSUPPORTED, L.DWARF_ERR_WORKSPACE
    assert all(fn(None, None) == bad for fn in (lib.dwarf_selective_scan_fwd, lib.dwarf_selective_scan_bwd, lib.dwarf_selective_scan_step))
    a = scan_args(L)
    f = a.fwd
    shared = [("B", -1, bad), ("N", -1, bad), ("D", 0, bad), ("G", 0, bad), ("G", 3, bad), ("S", 0, bad), ("S", 65, no), ("dtype", 3, bad),
              ("D", 1 << 22, no), ("N", (1 << 24) + 1, no), ("A", None, bad), ("x", None, bad), ("delta", P + 1, bad), ("Bm", None, bad),
              ("Cm", P + 1, bad), ("gate", P + 1, bad)]
    far = [(n + "_stride", (6400, s), no) for n in ("x", "delta", "gate") for s in (-64, 1 << 22)]
    far += [(n + "_stride", (3200, s, 16), no) for n in ("B", "C") for s in (-32, 1 << 22)]
    refused(lib.dwarf_selective_scan_fwd, f, shared + far + [
        ("y", None, bad), ("y_stride", (6400, 1 << 22), no), ("workspace", None, ws), ("B", 0, L.DWARF_OK), ("N", 0, L.DWARF_OK)])
    refused(lib.dwarf_selective_scan_bwd, a, shared + far, f)
    f.checkpoints, f.checkpoint_bytes = P, lib.dwarf_selective_scan_checkpoint_bytes(ctypes.byref(f)) - 1
    refused(lib.dwarf_selective_scan_fwd, f, [("checkpoints", P, ws)])
    refused(lib.dwarf_selective_scan_bwd, a, [("dy", P, ws)])
    f.checkpoint_bytes += 1
    refused(lib.dwarf_selective_scan_bwd, a, [
        ("dy", None, bad), ("dx", None, bad), ("ddelta", None, bad), ("dgate", None, bad), ("dB", None, bad), ("dC", P + 1, bad),
        ("dy_stride", (6400, 1 << 22), no), ("dx_stride", (6400, -64), no), ("ddelta_stride", (6400, 1 << 22), no),
        ("dgate_stride", (6400, 1 << 22), no), ("workspace", None, ws)])
    need = lib.dwarf_selective_scan_bwd_workspace_bytes(ctypes.byref(a))
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.dwarf_selective_scan_bwd(ctypes.byref(a), None) == ws
    a.workspace, a.workspace_bytes = P + 4, need
    assert lib.dwarf_selective_scan_bwd(ctypes.byref(a), None) == ws
    f.B, f.N = 1 << 10, 1 << 14   # the token sums' threads
    f.checkpoint_bytes = lib.dwarf_selective_scan_checkpoint_bytes(ctypes.byref(f))
    assert lib.dwarf_selective_scan_bwd(ctypes.byref(a), None) == no
    f.B = 1 << 23
    assert lib.dwarf_selective_scan_fwd(ctypes.byref(f), None) == no
    s = L.SelectiveScanStepArgs()
    s.R, s.D, s.G, s.S, s.pool, s.dtype = 3, 64, 2, 16, 5, L.DWARF_BF16
    s.x = s.delta = s.gate = s.Bm = s.Cm = s.A = s.out = s.state = s.new_state = P
    s.slot_stride = 64 * 16
    refused(lib.dwarf_selective_scan_step, s, [
        ("R", -1, bad), ("D", 0, bad), ("G", 3, bad), ("S", 65, no), ("S", 0, bad), ("dtype", 3, bad), ("R", 1 << 30, no), ("A", None, bad),
        ("x", None, bad), ("delta", P + 1, bad), ("Bm", None, bad), ("Cm", None, bad), ("gate", P + 1, bad), ("out", None, bad),
        ("state", P + 2, bad), ("new_state", None, bad), ("slot_stride", 64 * 16 - 1, bad), ("new_state", P + 64, bad), ("pool", 2, bad),
        ("R", 0, L.DWARF_OK)])


def test_checkpoints_of_gradients_that_cannot_be_formed_are_refused(pkg, lib):
    """The forward refuses what the backward would: before it has run, where it is asked for checkpoints."""
    L = pkg._lib
    a = scan_args(L)
    f = a.fwd
    f.B, f.N = 1 << 10, 1 << 14
    f.checkpoints, f.checkpoint_bytes = P, lib.dwarf_selective_scan_checkpoint_bytes(ctypes.byref(f))
    for fn, args in ((lib.dwarf_selective_scan_fwd, f), (lib.dwarf_selective_scan_bwd, a)):
        assert fn(ctypes.byref(args), None) == L.DWARF_ERR_UNSUPPORTED
        assert b"gradients" in lib.dwarf_last_error()


@pytest.mark.parametrize("S", [1, 8, 9, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("N", [1, 7, 8, 33, 257])
def test_checkpoint_sizes_agree(pkg, lib, N, S):
    """The fake tensors' size, computed in Python, is the library's."""
    f = scan_args(pkg._lib).fwd
    f.N, f.S = N, S
    assert 4 * pkg.selscan.checkpoint_elements(2, N, 64, S) == lib.dwarf_selective_scan_checkpoint_bytes(ctypes.byref(f))


@pytest.mark.parametrize("N", [(1 << 24) + 1, (1 << 31) - 1])
def test_sizes_of_refused_calls_are_zero(pkg, lib, N):
    """Token counts that the calls refuse, to the last that an int holds: no sizes are computed for them."""
    a = scan_args(pkg._lib)
    a.fwd.N = N
    f, b = ctypes.byref(a.fwd), ctypes.byref(a)
    assert lib.dwarf_selective_scan_checkpoint_bytes(f) == lib.dwarf_selective_scan_fwd_workspace_bytes(f) == 0
    assert lib.dwarf_selective_scan_bwd_workspace_bytes(b) == 0
    c = pkg._lib.CausalConvBwdArgs()
    c.fwd.B, c.fwd.N, c.fwd.D, c.fwd.W, c.fwd.dtype, c.dweight = 2, N, 64, 4, pkg._lib.DWARF_BF16, P
    assert lib.dwarf_causal_conv_bwd_workspace_bytes(ctypes.byref(c)) == 0


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def rejects(match, fn, *args, error=ValueError, **kw):
    with pytest.raises(error, match=match):
        fn(*args, **kw)


def test_norm_calls_refuse(pkg):
    for fn in (pkg.rms_norm, pkg.rms_norm_fp8):
        x = t(3, 4, 8)
        rejects("eps", fn, x, eps=-1.0)
        rejects("last dimension", fn, t(3, 0))
        rejects("weight must hold", fn, x, t(9))
        rejects("weight must hold", fn, x, t(3, 8))
        rejects("floating", fn, x, torch.zeros(8, dtype=torch.int32))
        rejects("bf16, fp16 or fp32", fn, x.double())
        rejects("residual", fn, x, residual=t(3, 8))
        rejects("residual", fn, x, residual=t(3, 4, 8, dtype=torch.float16))
        rejects("device tensors", fn, x, error=RuntimeError)


def test_conv_calls_refuse(pkg):
    x, w = t(2, 5, 8), t(8, 4)
    conv, step = pkg.causal_conv, pkg.causal_conv_step
    rejects("activation", conv, x, w, activation="relu")
    rejects("B,N,D", conv, t(5, 8), w)
    rejects("weight", conv, x, t(7, 4))
    rejects("weight", conv, x, torch.zeros(8, 4, dtype=torch.int64))
    rejects("8", conv, x, t(8, 9), error=(ValueError, RuntimeError))
    rejects("bias", conv, x, w, t(7))
    rejects("initial_state", conv, x, w, initial_state=t(2, 4, 8))
    rejects("initial_state", conv, x, w, initial_state=t(2, 3, 8, dtype=torch.float32))
    rejects("lengths", conv, x, w, lengths=torch.zeros(3, dtype=torch.int32))
    rejects("lengths", conv, x, w, lengths=torch.zeros(2))
    rejects("device tensors", conv, x, w, error=RuntimeError)
    row, pool = t(3, 8), t(5, 3, 8)
    rejects("activation", step, row, w, None, pool, activation="relu")
    rejects("pool", step, row, w, None, t(5, 4, 8))
    rejects("pool", step, row, w, None, t(5, 3, 16)[..., ::2])
    rejects("does not hold", step, row, w, None, t(2, 3, 8))
    rejects("slots", step, row, w, None, pool, slots=torch.zeros(2, dtype=torch.int32))
    rejects("new_state", step, row, w, None, pool, new_state=t(4, 3, 8))
    rejects("device tensors", step, row, w, None, pool, error=RuntimeError)


def test_scan_calls_refuse(pkg):
    f32 = torch.float32
    x, A, B = t(2, 5, 8), t(8, 4), t(2, 5, 2, 4)
    scan, step = pkg.selective_scan, pkg.selective_scan_step
    rejects("B,N,D", scan, t(5, 8), t(5, 8), A, B, B)
    rejects("delta", scan, x, t(2, 4, 8), A, B, B)
    rejects("delta", scan, x, x.float(), A, B, B)
    rejects("gate", scan, x, x, A, B, B, gate=t(2, 5, 7))
    rejects("A must", scan, x, x, t(7, 4), B, B)
    rejects("A must", scan, x, x, torch.zeros(8, 4, dtype=torch.int32), B, B)
    rejects("B must", scan, x, x, A, t(2, 5, 2, 5), B)
    rejects("C must", scan, x, x, A, B, B.float())
    rejects("share a shape", scan, x, x, A, B, t(2, 5, 4))
    rejects("divisible", scan, x, x, A, t(2, 5, 3, 4), t(2, 5, 3, 4))
    rejects("64 states", scan, x, x, t(8, 65), t(2, 5, 65), t(2, 5, 65), error=RuntimeError)
    rejects("skip", scan, x, x, A, B, B, skip=t(7))
    rejects("delta_bias", scan, x, x, A, B, B, delta_bias=torch.zeros(8, dtype=torch.int32))
    rejects("bf16, fp16 or fp32", scan, x.double(), x.double(), A, B.double(), B.double())
    rejects("device tensors", scan, x, x, A, B, B, error=RuntimeError)
    row, rb, pool = t(3, 8), t(3, 2, 4), t(5, 8, 4, dtype=f32)
    rejects("pool", step, row, row, A, rb, rb, pool.bfloat16())
    rejects("pool", step, row, row, A, rb, rb, t(5, 4, 8, dtype=f32).transpose(1, 2))
    rejects("does not hold", step, row, row, A, rb, rb, t(2, 8, 4, dtype=f32))
    rejects("slots", step, row, row, A, rb, rb, pool, slots=torch.zeros(3))
    rejects("new_state", step, row, row, A, rb, rb, pool, new_state=t(5, 8, 8, dtype=f32)[..., :4])
    rejects("device tensors", step, row, row, A, rb, rb, pool, error=RuntimeError)


@pytest.mark.parametrize("grouped", [False, True])
def test_fake_shapes(pkg, grouped):
    """Outputs of calls on fake device tensors: shapes and types."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda", requires_grad=True)   # noqa: E731
        x, A, Bm = e(2, 70, 48), e(48, 12, dtype=torch.float32), e(*((2, 70, 3, 12) if grouped else (2, 70, 12)))
        initial, gate, skip = e(2, 48, 12, dtype=torch.float32), e(2, 70, 48), e(48)
        y, s = pkg.selective_scan(x, x, A, Bm, Bm, skip=skip, gate=gate, initial_state=initial, return_state=True)
        assert y.requires_grad and s.requires_grad
        assert y.shape == x.shape and y.dtype == x.dtype and s.shape == (2, 48, 12) and s.dtype == torch.float32
        w, c, front = e(48, 4), e(48), e(2, 3, 48)
        y, s = pkg.causal_conv(x, w, c, activation="silu", initial_state=front, return_state=True)
        assert y.shape == x.shape and s.shape == (2, 3, 48) and s.dtype == x.dtype
        r = e(2, 70, 48, dtype=torch.float32)
        y, s = pkg.rms_norm(x, c, residual=r)
        assert y.dtype == x.dtype and s.dtype == torch.float32 and y.shape == s.shape == x.shape
        with torch.no_grad():
            q, scale, s = pkg.rms_norm_fp8(x, c, residual=r)
            assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (2, 70, 1)
            pool = e(5, 48, 12, dtype=torch.float32)
            assert pkg.selective_scan_step(x[:, 0], x[:, 0], A, Bm[:, 0], Bm[:, 0], pool).shape == (2, 48)
            assert pkg.causal_conv_step(x[:, 0], w, c, e(5, 3, 48)).shape == (2, 48)
