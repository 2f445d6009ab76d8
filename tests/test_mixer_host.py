"""Host side of the mixer's operators, without a GPU: the header's exports and layouts, refusals of bad calls, the
plan of rotary positions, the segment rule, fake shapes."""

import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from tests.conftest import ROOT

HEADER = os.path.join(ROOT, "include", "dwarf_mixer.h")
STRUCTS = {"dwarf_layer_norm_fwd_args": "LayerNormFwdArgs", "dwarf_layer_norm_bwd_args": "LayerNormBwdArgs",
           "dwarf_rotary_args": "RotaryArgs", "dwarf_linear_attention_fwd_args": "LinearAttentionFwdArgs",
           "dwarf_linear_attention_bwd_args": "LinearAttentionBwdArgs",
           "dwarf_linear_attention_step_args": "LinearAttentionStepArgs"}


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg._lib.load()


def test_header_exports_and_layout(pkg, lib, tmp_path):
    names = sorted(set(re.findall(r"^(?:int|int32_t|size_t)\s+(dwarf_\w+)\s*\(", open(HEADER).read(), re.M)))
    assert sorted(pkg._lib.MIXER_SYMBOLS) == names
    assert all(hasattr(lib, n) for n in names)
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dwarf_mixer.h"', "int main(void) {",
             'printf("f16 %d\\n", DWARF_F16);']
    for cname, pyname in STRUCTS.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in getattr(pkg._lib, pyname)._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out[0] == f"f16 {pkg._lib.DWARF_F16}"
    for line in out[1:]:
        cname, field, value = line.split()
        struct = getattr(pkg._lib, STRUCTS[cname])
        assert (ctypes.sizeof(struct) if field == "sizeof" else getattr(struct, field).offset) == int(value), line


P = 0x10000   # an aligned address that no refused call reads


def test_layer_norm_entry_points_refuse(pkg, lib):
    L = pkg._lib
    bad = L.DWARF_ERR_INVALID_ARGUMENT
    assert lib.dwarf_layer_norm_fwd(None, None) == bad and lib.dwarf_layer_norm_bwd(None, None) == bad
    a = L.LayerNormBwdArgs()
    f = a.fwd
    f.rows, f.groups, f.D, f.dtype, f.eps = 6, 1, 64, L.DWARF_BF16, 1e-5
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == bad           # x is NULL
    f.x, f.x_stride = P, (64, 64)
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == bad           # y is NULL
    f.x = P + 1
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == bad           # between elements
    f.x = P
    for name, value in (("D", 0), ("groups", 0), ("rows", -1), ("dtype", 7), ("eps", -1.0), ("eps", math.nan),
                        ("eps", math.inf)):
        keep = getattr(f, name)
        setattr(f, name, value)
        assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == bad, name
        assert lib.dwarf_layer_norm_bwd_workspace_bytes(ctypes.byref(a)) == 0
        setattr(f, name, keep)
    f.groups = 65536
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == L.DWARF_ERR_UNSUPPORTED
    f.groups, f.D = 1, (1 << 24) + 1
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == L.DWARF_ERR_UNSUPPORTED
    f.D = 64
    assert lib.dwarf_layer_norm_bwd(ctypes.byref(a), None) == bad           # dy is NULL
    a.dy, a.dy_stride, a.dweight = P, (64, 64), P
    need = lib.dwarf_layer_norm_bwd_workspace_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.dwarf_layer_norm_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.dwarf_layer_norm_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    f.rows = 0
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(f), None) == L.DWARF_OK    # nothing to do


def test_rotary_entry_point_refuses(pkg, lib):
    L = pkg._lib
    bad = L.DWARF_ERR_INVALID_ARGUMENT
    assert lib.dwarf_rotary(None, None) == bad
    a = L.RotaryArgs()
    a.B, a.H, a.H_kv, a.N, a.D, a.pairs, a.position_bytes, a.magnitude = 1, 2, 2, 4, 64, 32, 8, 1.0
    assert lib.dwarf_rotary(ctypes.byref(a), None) == bad                   # no positions
    a.positions = a.turns = P
    assert lib.dwarf_rotary(ctypes.byref(a), None) == bad                   # q is NULL
    a.q = a.q_out = P
    a.q_stride = a.q_out_stride = (512, 256, 64, 2)
    assert lib.dwarf_rotary(ctypes.byref(a), None) == bad                   # strided elements
    a.q_stride = (512, 256, 65, 1)
    a.q_out_stride, a.interleaved = (512, 256, 64, 1), 1
    assert lib.dwarf_rotary(ctypes.byref(a), None) == bad                   # odd strides, pairs side by side
    assert b"even strides" in lib.dwarf_last_error()
    a.q_stride = (512, 256, 64, 1)
    for name, value in (("D", 63), ("D", 0), ("pairs", 0), ("pairs", 33), ("dtype", 3), ("position_bytes", 2),
                        ("magnitude", math.nan), ("H", 0), ("N", -1)):
        keep = getattr(a, name)
        setattr(a, name, value)
        assert lib.dwarf_rotary(ctypes.byref(a), None) == bad, name
        setattr(a, name, keep)
    a.k, a.H_kv = P, 0
    assert lib.dwarf_rotary(ctypes.byref(a), None) == bad
    a.H_kv, a.B, a.N = 2, 1 << 20, 1 << 20
    assert lib.dwarf_rotary(ctypes.byref(a), None) == L.DWARF_ERR_UNSUPPORTED
    a.N = 0
    assert lib.dwarf_rotary(ctypes.byref(a), None) == L.DWARF_OK


def test_linear_attention_entry_points_refuse(pkg, lib):
    L = pkg._lib
    bad = L.DWARF_ERR_INVALID_ARGUMENT
    assert lib.dwarf_linear_attention_fwd(None, None) == bad and lib.dwarf_linear_attention_bwd(None, None) == bad
    assert lib.dwarf_linear_attention_step(None, None) == bad
    a = L.LinearAttentionBwdArgs()
    f = a.fwd
    f.B, f.H, f.H_kv, f.N, f.head_dim, f.scale = 2, 4, 2, 100, 64, 0.125
    rows, kv = (100 * 256, 64, 256, 1), (100 * 128, 64, 128, 1)
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == bad     # log_decay is NULL
    f.log_decay = P
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == bad     # q is NULL
    f.q = f.k = f.v = f.out = P
    f.q_stride = f.out_stride = rows
    f.k_stride = f.v_stride = kv
    need = lib.dwarf_linear_attention_states_bytes(ctypes.byref(f))
    assert need == 2 * 4 * 2 * 64 * 64 * 4                                  # two segments of 64
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == L.DWARF_ERR_WORKSPACE
    f.states, f.states_bytes = P, need - 1
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == L.DWARF_ERR_WORKSPACE
    f.states_bytes = need
    for name, value, want in (("H_kv", 3, bad), ("H_kv", 0, bad), ("head_dim", 128, L.DWARF_ERR_UNSUPPORTED),
                              ("dtype", 9, bad), ("scale", math.inf, bad), ("N", -1, bad), ("B", -1, bad),
                              ("N", (1 << 24) + 1, L.DWARF_ERR_UNSUPPORTED), ("q", P + 8, bad)):
        keep = getattr(f, name)
        setattr(f, name, value)
        assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == want, name
        assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == want, name
        setattr(f, name, keep)
    for stride in (0, 56, 1 << 22):                                         # overlapping rows, rows too far apart
        f.q_stride = (100 * 256, 64, stride, 1)
        assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == L.DWARF_ERR_UNSUPPORTED, stride
    f.q_stride = rows
    f.initial = P + 4
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == bad     # the state that enters is not aligned
    f.initial = None
    assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == bad     # dout is NULL
    a.dout = a.dq = a.dk = a.dv = a.dlog_decay = a.dfinal = P
    a.dout_stride = a.dq_stride = rows
    a.dk_stride = a.dv_stride = kv
    assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == bad     # the final state is needed
    for name in ("dfinal", "dinitial"):
        setattr(a, name, P + 8)
        assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == bad, name
        setattr(a, name, None)
    f.final = P + 8
    assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == bad
    f.final = None
    assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == L.DWARF_ERR_WORKSPACE
    s = L.LinearAttentionStepArgs()
    s.S, s.H, s.H_kv, s.pool, s.head_dim, s.scale = 3, 4, 2, 5, 64, 0.125
    s.q = s.k = s.v = s.out = s.log_decay = s.state = s.new_state = P
    s.q_stride = s.out_stride = (256, 64, 1)
    s.k_stride = s.v_stride = (128, 64, 1)
    s.slot_stride = 4 * 4096
    for name, value in (("slot_stride", 4 * 4096 - 4), ("slot_stride", 4 * 4096 + 2), ("pool", 2), ("pool", -1),
                        ("state", P + 4), ("new_state", P + 16), ("new_state", None), ("q", None), ("H_kv", 3),
                        ("scale", math.nan), ("S", -1)):
        keep = getattr(s, name)
        setattr(s, name, value)
        assert lib.dwarf_linear_attention_step(ctypes.byref(s), None) == bad, name
        setattr(s, name, keep)
    s.S = 0
    assert lib.dwarf_linear_attention_step(ctypes.byref(s), None) == L.DWARF_OK


def test_sizes_that_no_launch_holds_are_refused(pkg, lib):
    """Before anything is read or launched: more threads than 32 bits count."""
    L = pkg._lib
    a = L.LinearAttentionBwdArgs()
    f = a.fwd
    f.H, f.H_kv, f.head_dim, f.scale = 4, 2, 64, 0.125
    for B, N in ((1 << 21, 1), (1 << 20, 1025), (1 << 13, 1 << 18), (1 << 20, 0)):
        f.B, f.N = B, N
        assert lib.dwarf_linear_attention_fwd(ctypes.byref(f), None) == L.DWARF_ERR_UNSUPPORTED, (B, N)
        assert lib.dwarf_linear_attention_bwd(ctypes.byref(a), None) == L.DWARF_ERR_UNSUPPORTED, (B, N)
    s = L.LinearAttentionStepArgs()
    s.S, s.H, s.H_kv, s.head_dim, s.scale = 1 << 22, 4, 2, 64, 0.125
    assert lib.dwarf_linear_attention_step(ctypes.byref(s), None) == L.DWARF_ERR_UNSUPPORTED
    n = L.LayerNormFwdArgs()
    n.rows, n.groups, n.D, n.dtype, n.eps = 1, 1 << 9, 1 << 16, L.DWARF_BF16, 1e-5
    assert lib.dwarf_layer_norm_fwd(ctypes.byref(n), None) == L.DWARF_ERR_UNSUPPORTED


def test_step_refuses_out_in_its_inputs_memory(pkg):
    q, k, v = (torch.zeros(3, 4, 64) for _ in range(3))
    pool = torch.zeros(3, 4, 64, 64)
    for out in (q, v, pool[0, :3], torch.zeros(1, 4, 64).expand(3, 4, 64)):
        out = out if out.shape == q.shape else out.reshape(-1)[:768].view(3, 4, 64)
        with pytest.raises(ValueError, match="memory|aligned"):
            pkg.linear_attention_step(q, k, v, torch.zeros(4), pool, out=out)
    other = torch.zeros(3, 4, 64, 64)
    with pytest.raises(ValueError, match="new_state"):
        pkg.linear_attention_step(q, k, v, torch.zeros(4), pool, new_state=other, out=other.reshape(-1)[:768].view(3, 4, 64))


def test_step_refuses_out_among_rows_that_are_read(pkg):
    """Strided slices of one buffer: out is refused where it holds an element of another tensor, or one of its own twice,
    and accepted between them.  The truth is the set of the elements."""
    import random
    rng = random.Random(3)
    buf, pool, lg = torch.zeros(1 << 15), torch.zeros(2, 4, 64, 64), torch.zeros(4)
    at = (buf.data_ptr() // 4) % 4   # keeps every view 16-byte aligned

    def view(H, S=3):
        s1 = rng.choice([64, 64, 128, 192, 256, 72, 0, 20])
        s0 = rng.choice([64 * 12, 64 * 12, 64 * 12, 64 * 4, 64, 1024, 0, 200])
        return buf.as_strided((S, H, 64), (s0, s1, 1), (4 - at) % 4 + 4 * rng.randint(0, 256))

    def elements(t):
        S, H, _ = t.shape
        return [t.storage_offset() + s * t.stride(0) + h * t.stride(1) + d for s in range(S) for h in range(H) for d in range(64)]

    seen = set()
    for _ in range(600):
        S = rng.choice([1, 2, 3])
        tensors = dict(out=view(4, S), q=view(4, S), k=view(2, S), v=view(2, S))
        own = elements(tensors["out"])
        if len(set(own)) < len(own):
            want = "out"
        else:
            want = next((n for n in "qkv" if not set(own).isdisjoint(elements(tensors[n]))), None)
        seen.add(want)
        with pytest.raises((ValueError, RuntimeError)) as e:
            pkg.linear_attention_step(tensors["q"], tensors["k"], tensors["v"], lg, pool, slots=torch.zeros(S, dtype=torch.int32),
                                      out=tensors["out"])
        text = str(e.value)
        assert (f"shares memory with {want}" if want else "device tensors") in text, (want, text, tensors)
    assert seen == {"out", "q", "k", "v", None}
    fused = torch.zeros(3, 10, 64)   # out, q, k and v side by side in each row: allowed
    with pytest.raises(RuntimeError, match="device tensors"):
        pkg.linear_attention_step(fused[:, 4:8], fused[:, 8:9], fused[:, 9:], lg, torch.zeros(3, 4, 64, 64), out=fused[:, :4])
    layers = torch.zeros(3, 2, 4, 64, 64)   # out in a slot of the pool, and between the pool's slots
    rows = torch.zeros(3, 4, 64)
    for layer, want in ((0, "shares memory with state"), (1, "device tensors")):
        out = layers[:, layer, 0, :4]
        with pytest.raises((ValueError, RuntimeError), match=want):
            pkg.linear_attention_step(rows, rows, rows, lg, layers[:, 0], out=out)


def test_segment_rule_is_the_librarys(pkg, lib):
    for B in (1, 2, 3, 15, 20, 64):
        for H in (1, 6, 8, 32):
            for N in (1, 63, 64, 65, 777, 2048, 8192, 65536):
                seg = pkg.linattn.segment_tokens(B, H, N)
                assert seg == lib.dwarf_linear_attention_segment(B, H, N)
                a = pkg._lib.LinearAttentionFwdArgs()
                a.B, a.H, a.H_kv, a.N, a.head_dim = B, H, H, N, 64
                want = pkg.linattn.states_shape(B, H, N)
                assert lib.dwarf_linear_attention_states_bytes(ctypes.byref(a)) == 4 * math.prod(want)


def _qkv(S=(2, 4, 5, 64), Hkv=2, dtype=torch.bfloat16):
    kv = (S[0], Hkv, *S[2:])
    return torch.zeros(S, dtype=dtype), torch.zeros(kv, dtype=dtype), torch.zeros(kv, dtype=dtype)


def test_python_calls_refuse(pkg):
    q, k, v = _qkv()
    lg = torch.zeros(4)
    with pytest.raises(RuntimeError, match="device tensors"):
        pkg.linear_attention(q, k, v, lg)
    for args, kw in (((q[0], k, v, lg), {}), ((q, k, v[:, :1], lg), {}), ((q, k.float(), v, lg), {}),
                     ((q, k[:, :, :3], v[:, :, :3], lg), {}), ((q[:, :3], k, v, lg[:3]), {}), ((q, k, v, lg[:2]), {}),
                     ((q, k, v, lg.int()), {}), ((q.double(), k.double(), v.double(), lg), {}),
                     ((q, k, v, lg), dict(scale=math.inf)), ((q, k, v, lg), dict(initial_state=torch.zeros(2, 2, 64, 64))),
                     ((q, k, v, lg), dict(initial_state=torch.zeros(2, 4, 64, 64).bfloat16())),
                     ((q, k, v, lg), dict(lengths=torch.zeros(3, dtype=torch.int32))),
                     ((q, k, v, lg), dict(lengths=torch.zeros(2)))):
        with pytest.raises(ValueError):
            pkg.linear_attention(*args, **kw)
    q, k, v = (x[:, :, 0] for x in (q, k, v))
    pool = torch.zeros(3, 4, 64, 64)
    with pytest.raises(RuntimeError, match="device tensors"):
        pkg.linear_attention_step(q, k, v, lg, pool)
    for state, kw in ((pool.bfloat16(), {}), (pool[:, :2], {}), (pool[:1], {}), (pool.transpose(2, 3), {}),
                      (pool, dict(new_state=torch.zeros(4, 4, 64, 64))), (pool, dict(slots=torch.zeros(2))),
                      (pool, dict(slots=torch.zeros(3, dtype=torch.int32))), (pool, dict(scale=math.nan)),
                      (pool, dict(out=torch.zeros(2, 4, 64)))):
        with pytest.raises(ValueError):
            pkg.linear_attention_step(q, k, v, lg, state, **kw)
    x = torch.zeros(3, 4, 8)
    with pytest.raises(RuntimeError, match="device tensors"):
        pkg.layer_norm(x)
    for args in ((x, torch.zeros(4)), (x, torch.zeros(3, 8)), (x, torch.zeros(8), torch.zeros(4, 8)),
                 (x, torch.zeros(8, dtype=torch.int32)), (x, None, None, -1.0), (x, None, None, math.nan), (x.double(),),
                 (x.long(),), (torch.zeros(()),), (torch.zeros(3, 0),), (x, torch.zeros(3, 4, 8))):
        with pytest.raises(ValueError):
            pkg.layer_norm(*args)
    plan = pkg.rotary_plan(64, device="cpu")
    q, k, _ = _qkv()
    pos = torch.arange(5)
    with pytest.raises(RuntimeError, match="device tensors"):
        pkg.rotary_embed(q, k, pos, plan)
    for args in ((q[0], k, pos, plan), (q, k[:, :, :3], pos, plan), (q, k.float(), pos, plan), (q, k, pos[:4], plan),
                 (q, k, pos.float(), plan), (q, k, pos.expand(3, 5), plan), (q[..., :32], k[..., :32], pos, plan),
                 (q.double(), None, pos, plan), (q[..., :63], None, pos, pkg.rotary_plan(32, device="cpu"))):
        with pytest.raises(ValueError):
            pkg.rotary_embed(*args)


def test_custom_ops_refuse(pkg):
    """The custom ops are called without the Python checks of compiled calls too: their launches check for themselves."""
    ops = torch.ops.dwarf
    x, w = torch.zeros(3, 4, 8), torch.zeros(4, 8)
    for args in ((x, None, None, 0, 1e-5), (x, None, None, 3, 1e-5), (x, w, None, 1, 1e-5), (x, None, w[:2], 4, 1e-5),
                 (x, w.int(), None, 4, 1e-5), (torch.zeros(3, 0), None, None, 1, 1e-5), (x.double(), None, None, 1, 1e-5)):
        with pytest.raises(ValueError):
            ops.layer_norm_fwd(*args)
    for args in ((x[:2], x, None, 1), (x, x, w, 1), (x, x, None, 0)):
        with pytest.raises(ValueError):
            ops.layer_norm_bwd(*args, 1e-5, True, True, True)
    q, k, v = _qkv()
    pos, turns = torch.arange(5), torch.zeros(32, dtype=torch.int64)
    for args in ((q, k[:, :, :3], pos, turns), (q, k, pos[:4], turns), (q, k, pos, turns.int()), (q, k, pos, turns.repeat(2)),
                 (q, k, pos, torch.zeros(64, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError):
            ops.rotary(*args, False, False, 1.0)
    lg, state, states = torch.zeros(4), torch.zeros(2, 4, 64, 64), torch.zeros(0)
    for args in ((q, k[:, :, :3], v[:, :, :3], lg, None, None), (q, k, v, lg[:2], None, None), (q, k, v, lg, state[:1], None),
                 (q, k, v, lg, None, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.linear_attention_fwd(*args, 0.125, True)
        with pytest.raises(ValueError):
            ops.linear_attention_bwd(q, None, *args, 0.125, states, None, True, True)
    for dout, dstate, st, kept in ((q[:, :, :3], None, states, None), (q, state[:1], states, None), (q, None, states.int(), None),
                                   (q, None, states, state[:, :2]), (q, None, states, state.transpose(2, 3))):
        with pytest.raises(ValueError):
            ops.linear_attention_bwd(dout, dstate, q, k, v, lg, None, None, 0.125, st, kept, True, True)
    q, k, v = (x[:, :, 0] for x in (q, k, v))
    for pool, slots in ((state[:1], None), (state.bfloat16(), None), (state, torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.linear_attention_step_(q, k, v, lg, pool, slots, 0.125)
        with pytest.raises(ValueError):
            ops.linear_attention_step(q, k, v, lg, pool, pool.clone(), slots, 0.125)
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.linear_attention_step_(q, k, v, lg, state, None, 0.125)


def _tangent_calls(pkg, tensors):
    """(name, call) for each floating tensor of each operator, the tensor taken from ``tensors`` (name -> tensor)."""
    t = tensors
    args = (t["q"], t["k"], t["v"], t["log_decay"])
    rows = tuple(t[n][:, :, 0] for n in ("q", "k", "v"))
    return (("layer_norm", lambda: pkg.layer_norm(t["x"], t["weight"], t["bias"]), ("x", "weight", "bias")),
            ("rotary_embed", lambda: pkg.rotary_embed(t["q"], t["k"], t["positions"], t["plan"]), ("q", "k")),
            ("linear_attention", lambda: pkg.linear_attention(*args, initial_state=t["initial"]),
             ("q", "k", "v", "log_decay", "initial")),
            ("linear_attention_step", lambda: pkg.linear_attention_step(*rows, t["log_decay"], t["pool"]),
             ("q", "k", "v", "log_decay", "pool")),
            ("layer_norm", lambda: torch.ops.dwarf.layer_norm_fwd(t["x"], t["weight"], t["bias"], 1, 1e-5), ("x", "weight", "bias")),
            ("layer_norm", lambda: torch.ops.dwarf.layer_norm_bwd(t["x"], t["x"], t["weight"], 1, 1e-5, True, True, True),
             ("x", "weight")),
            ("rotary_embed", lambda: torch.ops.dwarf.rotary(t["q"], t["k"], t["positions"], t["plan"].turns, False, False, 1.0),
             ("q", "k")),
            ("linear_attention", lambda: torch.ops.dwarf.linear_attention_fwd(*args, t["initial"], None, 0.125, True),
             ("q", "k", "v", "log_decay", "initial")),
            ("linear_attention", lambda: torch.ops.dwarf.linear_attention_bwd(
                t["q"], t["initial"], *args, None, None, 0.125, t["states"], None, True, False), ("q", "k", "v", "log_decay", "initial")),
            ("linear_attention_step", lambda: torch.ops.dwarf.linear_attention_step_(*rows, t["log_decay"], t["pool"], None, 0.125),
             ("q", "k", "v", "log_decay", "pool")))


def test_forward_mode_derivatives_are_refused(pkg):
    """A tangent of any input, which the results would drop, is an error (before the device is asked for)."""
    import torch.autograd.forward_ad as fw
    q, k, v = _qkv(dtype=torch.float32)
    base = dict(q=q, k=k, v=v, log_decay=torch.zeros(4), initial=torch.zeros(2, 4, 64, 64), pool=torch.zeros(3, 4, 64, 64),
                x=torch.zeros(3, 8), weight=torch.ones(8), bias=torch.zeros(8), states=torch.zeros(0), positions=torch.arange(5),
                plan=pkg.rotary_plan(64, device="cpu"))
    count = len(_tangent_calls(pkg, base))
    for i in range(count):
        for name in _tangent_calls(pkg, base)[i][2]:
            with fw.dual_level():
                dual = dict(base, **{name: fw.make_dual(base[name], torch.ones_like(base[name]))})
                what, call, _ = _tangent_calls(pkg, dual)[i]
                with pytest.raises(RuntimeError, match=f"{what} has no derivative in forward mode"):
                    call()
    with pytest.raises(RuntimeError, match="has no derivative in forward mode"):
        torch.func.jvp(pkg.layer_norm, (base["x"],), (base["x"],))


def test_fake_tensors_give_shapes(pkg):
    """Tensors without memory, with and without gradients: the custom ops' shapes, as the other operators of the package
    give them, and no launch."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    plan = pkg.rotary_plan(64, device="cpu")
    with FakeTensorMode():
        make = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")   # noqa: E731
        for grad in (False, True):
            q, k = make(2, 4, 70, 64, dtype=torch.bfloat16), make(2, 2, 70, 64, dtype=torch.bfloat16)
            x, w, lg = make(3, 4, 8, dtype=torch.float16), make(4, 8), make(4)
            for t in (q, k, x, w, lg):
                t.requires_grad_(grad)
            plan.turns = make(32, dtype=torch.int64)
            qr, kr = pkg.rotary_embed(q, k, torch.arange(70, device="cuda"), plan)
            alone, none = pkg.rotary_embed(q, None, torch.arange(70, device="cuda"), plan)
            o, state = pkg.linear_attention(qr, kr, kr, lg, return_state=True)
            y = pkg.layer_norm(x, w, w)
            assert none is None and alone.shape == q.shape
            assert qr.shape == q.shape and kr.shape == k.shape and o.shape == q.shape and y.shape == x.shape
            assert state.shape == (2, 4, 64, 64) and state.dtype == torch.float32
            assert o.transpose(1, 2).is_contiguous() and qr.transpose(1, 2).is_contiguous()
            assert all(isinstance(t, FakeTensor) and t.requires_grad == grad for t in (qr, kr, o, state, y))
        pool, rows = make(5, 4, 64, 64), make(3, 4, 64, dtype=torch.bfloat16)
        out = make(3, 4, 64, dtype=torch.bfloat16)
        with torch.no_grad():
            one = pkg.linear_attention_step(rows, rows, rows, lg, pool, slots=make(3, dtype=torch.int64))
            assert one.shape == (3, 4, 64) and one.dtype == torch.bfloat16
            assert pkg.linear_attention_step(rows, rows, rows, lg, pool, new_state=make(5, 4, 64, 64), out=out) is out
            for bad in (make(3, 4, 64), make(2, 4, 64, dtype=torch.bfloat16)):
                with pytest.raises(ValueError, match="out must be"):
                    pkg.linear_attention_step(rows, rows, rows, lg, pool, out=bad)
        with pytest.raises(ValueError, match="floating"):
            pkg.layer_norm(x, make(8, dtype=torch.int32))


def test_traces_hold_the_operators(pkg):
    """make_fx records the custom ops, not an allocation that nothing writes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def layer(x, w, lg):
        y = pkg.layer_norm(x, w)
        q, k = pkg.rotary_embed(y.transpose(1, 2), None, positions, plan)[0], y.transpose(1, 2)
        o, state = pkg.linear_attention(q, k, k, lg, return_state=True)
        with torch.no_grad():
            one = pkg.linear_attention_step(q[:, :, 0], k[:, :, 0], k[:, :, 0], lg, state.clone())
        return [o, one]

    plan = pkg.rotary_plan(64, device="cpu")
    with FakeTensorMode():
        plan.turns, positions = torch.empty(32, dtype=torch.int64, device="cuda"), torch.arange(70, device="cuda")
        args = (torch.empty(2, 70, 4, 64, device="cuda", dtype=torch.bfloat16), torch.empty(4, 64, device="cuda"),
                torch.empty(4, device="cuda"))
        graph = make_fx(layer)(*args)
    seen = [str(n.target) for n in graph.graph.nodes]
    for name in ("layer_norm_fwd", "rotary", "linear_attention_fwd", "linear_attention_step_"):
        assert seen.count(f"dwarf.{name}.default") == 1, (name, seen)


def test_rotary_plan_frequencies(pkg):
    """Turns are the nearest 2^-64 fractions, and each scaling gives its formula's frequencies."""
    plan = pkg.rotary_plan(64, device="cpu")
    f = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert torch.equal(plan.inverse_frequencies, f)
    got = torch.tensor([(t % 2 ** 64) / 2 ** 64 for t in plan.turns.tolist()], dtype=torch.float64) * 2 * math.pi
    torch.testing.assert_close(got, f, rtol=4e-16, atol=1e-18)   # three float64 roundings
    lin = pkg.rotary_plan(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin.inverse_frequencies, f / 4)
    ntk = pkg.rotary_plan(64, scaling="base", factor=8.0, device="cpu").inverse_frequencies
    assert float(ntk[0]) == 1.0
    assert abs(float(ntk[-1] * 8 / f[-1]) - 1) < 1e-12   # the slowest pair is stretched by the factor
    bands = pkg.rotary_plan(64, scaling="bands", factor=16.0, original_length=2048, device="cpu").inverse_frequencies
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(bands[turns >= 32], f[turns >= 32])
    slow = turns <= 1
    assert slow.any() and torch.allclose(bands[slow], f[slow] / 16, rtol=1e-15)
    assert bool((bands[1:] < bands[:-1]).all())
    own = pkg.rotary_plan(6, inverse_frequencies=torch.tensor([1.0, -0.5, 0.0]), device="cpu")
    assert own.turns.tolist()[2] == 0 and own.turns.tolist()[1] < 0
    assert own.to("cpu").turns.tolist() == own.turns.tolist()
    for args, kw in (((7,), {}), ((0,), {}), ((64,), dict(scaling="other")), ((64,), dict(factor=0.0)),
                     ((64,), dict(base=-1.0)), ((64,), dict(scaling="bands", factor=2.0)),
                     ((64,), dict(scaling="bands", original_length=2048, fast_turns=1.0, slow_turns=2.0)),
                     ((2,), dict(scaling="base", factor=2.0)), ((64,), dict(magnitude=math.nan)),
                     ((64,), dict(inverse_frequencies=torch.ones(3))),
                     ((2,), dict(inverse_frequencies=torch.tensor([math.inf])))):
        with pytest.raises(ValueError):
            pkg.rotary_plan(*args, device="cpu", **kw)


def test_fake_shapes(pkg):
    m = torch.device("meta")
    q, k = torch.empty(2, 4, 300, 64, device=m, dtype=torch.bfloat16), torch.empty(2, 2, 300, 64, device=m, dtype=torch.bfloat16)
    lg = torch.empty(4, device=m)
    out, state, states = torch.ops.dwarf.linear_attention_fwd(q, k, k, lg, None, None, 0.125, True)
    assert out.shape == q.shape and out.transpose(1, 2).is_contiguous() and state.shape == (2, 4, 64, 64)
    assert states.shape == pkg.linattn.states_shape(2, 4, 300) and states.dtype == torch.float32
    g = torch.ops.dwarf.linear_attention_bwd(out, None, q, k, k, lg, state, None, 0.125, states, None, True, False)
    assert [tuple(x.shape) for x in g] == [tuple(q.shape), tuple(k.shape), tuple(k.shape), (4,), (0,)]
    a, b = torch.ops.dwarf.rotary(q, k, torch.empty(300, device=m, dtype=torch.int64),
                                  torch.empty(32, device=m, dtype=torch.int64), False, False, 1.0)
    assert a.shape == q.shape and b.shape == k.shape and b.transpose(1, 2).is_contiguous()
    x = torch.empty(3, 4, 8, device=m, dtype=torch.float16)
    w = torch.empty(4, 8, device=m)
    y = torch.ops.dwarf.layer_norm_fwd(x, w, w, 4, 1e-5)
    assert y.shape == x.shape and y.dtype == torch.float16
    dx, dw, db = torch.ops.dwarf.layer_norm_bwd(y, x, w, 4, 1e-5, True, True, False)
    assert dx.shape == x.shape and dw.shape == (32,) and db.shape == (0,)
    pool = torch.empty(5, 4, 64, 64, device=m)
    o = torch.ops.dwarf.linear_attention_step(q[:, :, 0], k[:, :, 0], k[:, :, 0], lg, pool, pool.clone(), None, 0.125)
    assert o.shape == (2, 4, 64)
