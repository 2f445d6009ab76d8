"""CPU restatement of the mixer's operators in float64 -- test infrastructure, not the product.

``linear_attention``: the recurrence S_t = g S_{t-1} + k_t v_t^T, o_t = scale q_t S_t token by token, with
g = exp(min(log_decay, 0)); ``linear_attention_backward``: its adjoint recurrence, token by token.
``linear_attention_chunked``: the same in blocks of tokens, for long sequences, its gradients by autograd.
``rotary``: each pair as a complex number times exp(i position f).  ``layer_norm`` and its gradients from the formula.
"""

from __future__ import annotations

import torch


def linear_attention(q, k, v, log_decay, scale, initial=None, lengths=None):
    """(out [B,H,N,D], state [B,H,D,D]) of q [B,H,N,D], k, v [B,Hkv,N,D]."""
    B, H, N, D = q.shape
    group = H // k.shape[1]
    out = torch.zeros(B, H, N, D, dtype=torch.float64)
    state = torch.zeros(B, H, D, D, dtype=torch.float64) if initial is None else initial.double().clone()
    g = torch.exp(log_decay.double().clamp(max=0))
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for t in range(n):
            kt, vt = (x[b, :, t].double().repeat_interleave(group, 0) for x in (k, v))
            state[b] = g[:, None, None] * state[b] + kt[:, :, None] * vt[:, None, :]
            out[b, :, t] = scale * torch.einsum("hd,hde->he", q[b, :, t].double(), state[b])
    return out, state


def linear_attention_backward(q, k, v, log_decay, scale, dout, initial=None, lengths=None, dstate=None):
    """(dq, dk, dv, dlog_decay [H], dinitial)."""
    B, H, N, D = q.shape
    Hkv = k.shape[1]
    group = H // Hkv
    g = torch.exp(log_decay.double().clamp(max=0))[:, None, None]
    dq = torch.zeros(B, H, N, D, dtype=torch.float64)
    dk, dv = (torch.zeros(B, H, N, D, dtype=torch.float64) for _ in range(2))
    dlog = torch.zeros(H, dtype=torch.float64)
    dinitial = torch.zeros(B, H, D, D, dtype=torch.float64)
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        S = torch.zeros(H, D, D, dtype=torch.float64) if initial is None else initial[b].double()
        before = []
        for t in range(n):
            kt, vt = (x[b, :, t].double().repeat_interleave(group, 0) for x in (k, v))
            before.append(S)
            S = g * S + kt[:, :, None] * vt[:, None, :]
            dq[b, :, t] = scale * torch.einsum("hde,he->hd", S, dout[b, :, t].double())
        G = torch.zeros(H, D, D, dtype=torch.float64) if dstate is None else dstate[b].double()
        for t in reversed(range(n)):
            kt, vt = (x[b, :, t].double().repeat_interleave(group, 0) for x in (k, v))
            G = G + scale * q[b, :, t].double()[:, :, None] * dout[b, :, t].double()[:, None, :]
            dk[b, :, t] = torch.einsum("hde,he->hd", G, vt)
            dv[b, :, t] = torch.einsum("hde,hd->he", G, kt)
            dlog += (G * g * before[t]).sum((-1, -2))
            G = g * G
        dinitial[b] = G
    dlog = torch.where(log_decay.double() > 0, torch.zeros((), dtype=torch.float64), dlog)
    shared = lambda x: x.reshape(B, Hkv, group, N, D).sum(2)   # noqa: E731
    return dq, shared(dk), shared(dv), dlog, dinitial


def linear_attention_chunked(q, k, v, log_decay, scale, dout, initial=None, lengths=None, dstate=None, block=64):
    """(out, state, (dq, dk, dv, dlog_decay, dinitial), crossing): crossing[b] holds <S, G> per head, the state behind
    every ``block`` tokens of sequence b (the first one: what enters) times its adjoint."""
    B, H, N, D = q.shape
    group = H // k.shape[1]
    leaves = [x.double().clone().requires_grad_(True) for x in (q, k, v, log_decay)]
    S0 = (torch.zeros(B, H, D, D, dtype=torch.float64) if initial is None else initial.double().clone()).requires_grad_(True)
    ql, kl, vl, lgl = leaves
    lg = lgl.clamp(max=0)[:, None, None]
    outs, ends, passed = [], [], []
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        S, rows, kept = S0[b], [], []
        for t in range(0, n, block):
            m = min(block, n - t)
            S = S * 1.0   # a value of its own, whose gradient is the adjoint here
            kept.append(S)
            i = torch.arange(m, dtype=torch.float64)
            gap = i[:, None] - i[None, :]
            near = torch.where(gap >= 0, torch.exp(lg * gap.clamp(min=0)), torch.zeros((), dtype=torch.float64))
            qb, kb, vb = ql[b, :, t:t + m], *(x[b, :, t:t + m].repeat_interleave(group, 0) for x in (kl, vl))
            rows.append(scale * ((qb @ kb.transpose(1, 2) * near) @ vb + torch.exp(lg * (i[:, None] + 1)) * (qb @ S)))
            S = torch.exp(lg * m) * S + (kb * torch.exp(lg * (m - 1 - i)[:, None])).transpose(1, 2) @ vb
        outs.append(torch.cat([*rows, torch.zeros(H, N - n, D, dtype=torch.float64)], 1))
        ends.append(S)
        passed.append(kept)
    out, state = torch.stack(outs), torch.stack(ends)
    loss = (out * dout.double()).sum() + (0 if dstate is None else (state * dstate.double()).sum())
    flat = [S for kept in passed for S in kept]
    grads = torch.autograd.grad(loss, [*leaves, S0, *flat], allow_unused=True)
    given = [torch.zeros_like(x) if g is None else g for x, g in zip([*leaves, S0], grads)]
    at, crossing = 5, []
    for kept in passed:
        crossing.append([(S.detach() * g).sum((1, 2)) for S, g in zip(kept, grads[at:at + len(kept)])])
        at += len(kept)
    return out.detach(), state.detach(), tuple(given), crossing


def rotary(x, positions, frequencies, interleaved, magnitude=1.0, inverse=False):
    """x [B,H,N,D] with its first 2 * len(frequencies) elements turned."""
    n = frequencies.numel()
    pos = positions.double()
    angle = (pos[:, None] if pos.ndim == 1 else pos[:, None, :, None]) * frequencies.double()
    turn = torch.polar(torch.full_like(angle, float(magnitude)), -angle if inverse else angle)
    y = x.double().clone()
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = z.real, z.imag
    else:
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    return y


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    x = x.double()
    centred = x - x.mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def layer_norm_backward(dy, x, weight=None, eps=1e-5):
    """(dx, dweight, dbias); dweight and dbias in the shape of the last dimension, or of weight."""
    x, g = x.double(), dy.double()
    centred = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    h = centred * r
    gw = g if weight is None else g * weight.double()
    dx = r * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    lead = tuple(range(x.ndim - (1 if weight is None else weight.ndim)))
    return dx, (g * h).sum(lead), g.sum(lead)
