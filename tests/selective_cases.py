"""Inputs and error bounds of the selective mixer's GPU tests.

Bounds are sums of what each rounding can do, in units of u = 2^-24 (half a step of fp32), next to the size of what is
rounded; ``within`` of mixer_cases adds the last rounding to the result's type.
"""

import math

import torch

from oracle import selective_ref
from tests import mixer_cases

U = 2.0 ** -24


def within(got, want, terms, dtype, slack):
    """mixer_cases' check, also of tensors without elements."""
    want = want.detach()
    assert got.shape == want.shape
    if want.numel():
        mixer_cases.within(got, want, terms.detach(), dtype, slack)


def f64(t):
    return None if t is None else t.detach().double().cpu()


def sigmoid_off(p):
    """1 / (1 + e^-p) relative: the exponent's argument is rounded and its factor is (1.25 |p|), exp2 and the reciprocal
    are within a step (2 each), the sum half a step, with half a step to spare."""
    return 1.25 * p.abs() + 6


def silu_off(p, p_off):
    """Absolute, of silu(p) whose p is p_off off: silu's slope is below 1.1."""
    return 1.1 * p_off + selective_ref.silu(p).abs() * (sigmoid_off(p) + 1)


def slope_off(p, p_off):
    """Absolute, of silu'(p) = e (1 + p (1 - e)): e is e (1.25 |p| + 6) off, 1 - e that and half a step, the products and the
    sum another three; its slope in p is below 0.5."""
    return (1 + 2 * p.abs()) * (sigmoid_off(p) + 4) + 0.5 * p_off


def segment_tokens(b, n, D, G, S):
    """Tokens of a segment, as the launches choose them, and whether there is more than one."""
    per, tile = D // G, 4 * (64 // (4 if S <= 32 else 8))
    groups = b * -(-per // tile) * G
    segs = 1 if groups >= 192 else min(512 // groups, 64)
    seg = max(-(--(-n // segs) // 32) * 32, 64)
    return seg, n > seg


def conv_strips(b, n, D, dtype):
    """Tokens of the convolution's strips forward and backward, as the launches choose them."""
    def strip(vec):
        blocks = -(-(-(-D // vec)) // 32)
        tokens = 16
        while tokens < 64 and b * n // (2 * tokens) // 8 * blocks >= 448:
            tokens *= 2
        return tokens
    per = 4 if dtype == torch.float32 else 8
    return strip(per if D >= per else 1), strip(4 if D >= 4 else 1)


def norm_grid(rows, groups, D, dtype, backward):
    """Workgroups of the norm's register kernels on aligned rows, and the rows of each, as the launches choose them."""
    per, threads = 4 if dtype == torch.float32 else 8, 512 if backward else 256
    units = D // per if D % per == 0 else D
    k = 1
    for tpr in (8, 16, 32, 64):
        if units <= tpr:
            break
    else:
        if units <= 256:
            k = 2 if units <= 128 else 4
        else:
            assert units <= 2048
            tpr = threads if units <= 4 * threads else 512
            k = 1 if units <= tpr else 2 if units <= 2 * tpr else 4
    each = threads // tpr if tpr < threads else 1
    most = 2048 if not backward else 256 if k >= 2 else 512
    unit = groups // math.gcd(groups, each)
    blocks = -(-min(-(-rows * groups // each), most) // unit) * unit
    return blocks, each


def scan_bounds(a, softplus, lengths=None, dy=None, dstate=None):
    """Bounds in u for y, state and, with dy, every gradient of the scan of a (a dict of float64 inputs)."""
    x, delta, A, B, C = (a[k] for k in ("x", "delta", "A", "B", "C"))
    skip, gate, bias, initial = (a.get(k) for k in ("skip", "gate", "delta_bias", "initial"))
    b, n, D = x.shape
    S = A.shape[1]
    grouped = B.ndim == 4
    G = B.shape[2] if grouped else 1
    if not grouped:
        B, C = B[:, :, None], C[:, :, None]
    per = D // G
    wide = lambda t: t.repeat_interleave(per, 1)   # noqa: E731  [b,G,S] to channels
    raw = delta if bias is None else delta + bias
    step = torch.nn.functional.softplus(raw) if softplus else raw
    alive = torch.ones(b, n, 1, dtype=torch.float64)
    if lengths is not None:
        alive = (torch.arange(n)[None] < lengths[:, None].clamp(0, n)).double()[..., None]
    step, u = step * alive, x * alive
    seg, several = segment_tokens(b, n, D, G, S)
    # the step: the sum delta + bias half a step of raw (which moves the softplus by at most its own part), the softplus
    # 3.5e-7 relative (6 u)
    st_off = (raw.abs() + 8) if softplus else torch.ones_like(raw)
    su = step * u
    # a = exp2(step rate): the argument's three roundings and the step's, relative to its size; where segments are joined
    # also the sum of a segment's steps, a chain of a quarter of its tokens; exp2 itself one step and the product half
    rate = (step[..., None] * A).abs()
    a_off = rate * (st_off[..., None] + 3 + (seg / 4 + 8 if several else 0)) + 3
    dec = torch.exp(step[..., None] * A)
    H = torch.zeros(b, D, S, dtype=torch.float64) if initial is None else initial.abs()
    h = torch.zeros_like(H) if initial is None else initial
    E = torch.zeros_like(H)
    act, act_off = torch.ones_like(x), torch.zeros_like(x)
    if gate is not None:
        act, act_off = selective_ref.silu(gate), silu_off(gate, torch.zeros_like(gate))
    k = torch.zeros(D, dtype=torch.float64) if skip is None else skip
    y_off, hs, Hs, Es = torch.zeros_like(x), [], [], []
    for t in range(n):
        add = (su[:, t, :, None] * wide(B[:, t])).abs()
        Hn = dec[:, t] * H + add
        E = dec[:, t] * E + dec[:, t] * H * a_off[:, t] + add * (st_off[:, t, :, None] + 2) + Hn * (2 if several else 1) * alive[:, t, :, None]
        hs.append(h), Hs.append(H), Es.append(E)   # h, H in front of the token, E behind it
        h = dec[:, t] * h + su[:, t, :, None] * wide(B[:, t])
        H = Hn
        Ct = wide(C[:, t]).abs()
        o_abs = (Ct * H).sum(-1) + (k * u[:, t]).abs()
        o_off = (Ct * E).sum(-1) + (S + 8) * o_abs
        y_off[:, t] = (act[:, t].abs() * (o_off + o_abs) + o_abs * act_off[:, t]) * alive[:, t]
    off = dict(y=y_off, state=E)
    if dy is None:
        return off
    dy = dy * alive
    do, do_off = (dy * act).abs(), dy.abs() * (act_off + act.abs())
    P = torch.zeros_like(H) if dstate is None else dstate.abs()   # |a_{t+1} g_{t+1}|
    EP = torch.zeros_like(P)
    z = torch.zeros_like
    off.update(x=z(x), delta=z(x), gate=z(x), A=z(A), B=z(B), C=z(C), skip=z(A[:, 0]), delta_bias=z(A[:, 0]))
    tiles = -(-per // 32) + 40   # sums over channels: lanes, waves, tiles
    sums = lambda t: t.view(b, G, per, S).sum(2)   # noqa: E731
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    slope_rel = sigmoid_off(raw) + raw.abs() + 1 if softplus else torch.zeros_like(raw)
    for t in reversed(range(n)):
        Bt, Ct, on = wide(B[:, t]).abs(), wide(C[:, t]).abs(), alive[:, t]
        Hn = dec[:, t] * Hs[t] + (su[:, t, :, None] * wide(B[:, t])).abs()
        En = Es[t]
        Ein = Es[t - 1] if t else z(En)
        g = Ct * do[:, t, :, None] + P
        Eg = Ct * do_off[:, t, :, None] + EP + g * (2 if several else 1) * on[..., None]
        so = st_off[:, t]
        into = (Bt * g).sum(-1)
        into_off = (Bt * Eg).sum(-1) + (S + 8) * into
        st, xt = step[:, t].abs(), u[:, t].abs()
        off["x"][:, t] = on * (st * into_off + st * into * (so + 2) + (k.abs() * (do_off[:, t] + 2 * do[:, t])))
        m = dec[:, t] * g * Hs[t]
        m_off = dec[:, t] * (Hs[t] * Eg + g * Ein) + m * (a_off[:, t] + 3)
        mA, mA_off = (m * A.abs()).sum(-1), (m_off * A.abs()).sum(-1)
        dd = xt * into + mA
        dd_off = xt * into_off + mA_off + (S + 12) * dd
        off["delta"][:, t] = on * slope[:, t] * (dd_off + dd * slope_rel[:, t])
        off["A"] += ((st[..., None] * (m_off + m * (so[..., None] + 34))) * on[..., None]).sum(0)
        off["B"][:, t] = sums(((st * xt)[..., None] * (Eg + g * (so[..., None] + 2 + tiles))) * on[..., None])
        off["C"][:, t] = sums((do[:, t, :, None] * En + Hn * (do_off[:, t, :, None] + do[:, t, :, None] * tiles)) * on[..., None])
        off["skip"] += (xt * (do_off[:, t] + 34 * do[:, t])).sum(0)
        off["delta_bias"] += (off["delta"][:, t] + 34 * slope[:, t] * dd * on).sum(0)
        if gate is not None:
            o_abs = (Ct * Hn).sum(-1) + (k * u[:, t]).abs()
            o_off = (Ct * En).sum(-1) + (S + 8) * o_abs
            e = torch.sigmoid(gate[:, t])
            sl = (e * (1 + gate[:, t] * (1 - e))).abs()
            off["gate"][:, t] = on * dy[:, t].abs() * (o_off * sl + o_abs * (slope_off(gate[:, t], z(e)) + 2 * sl))
        P, EP = dec[:, t] * g, dec[:, t] * (Eg + g * a_off[:, t]) + dec[:, t] * g
    off["initial"] = EP
    if not grouped:
        off["B"], off["C"] = off["B"][:, :, 0], off["C"][:, :, 0]
    return off
