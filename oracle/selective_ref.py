"""CPU restatement of the selective mixer's operators in float64 -- test infrastructure, not the product.

``selective_scan``: the recurrence token by token, every input a float64 tensor; its gradients come from autograd through
the same lines.  ``causal_conv``: the sum over the taps.  ``rms_norm``: the formula, the residual's sum rounded to the
stream's type as the definition says.
"""

from __future__ import annotations

import torch


def silu(z):
    return z / (1 + torch.exp(-z))


def selective_scan(x, delta, A, B, C, skip=None, gate=None, delta_bias=None, softplus=False, initial=None, lengths=None):
    """(y [B,N,D], state [B,D,S]) of x, delta [b,n,D], A [D,S], B, C [b,n,G,S] or [b,n,S], all float64."""
    b, n, D = x.shape
    if B.ndim == 3:
        B, C = B[:, :, None], C[:, :, None]
    per = D // B.shape[2]
    raw = delta if delta_bias is None else delta + delta_bias
    step = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw   # its slope is 1/2 at 0 too
    rows, states = [], []
    for i in range(b):
        count = n if lengths is None else min(max(int(lengths[i]), 0), n)
        h = x.new_zeros(D, A.shape[1]) if initial is None else initial[i]
        out = []
        for t in range(count):
            Bt, Ct = B[i, t].repeat_interleave(per, 0), C[i, t].repeat_interleave(per, 0)
            h = torch.exp(step[i, t, :, None] * A) * h + (step[i, t] * x[i, t])[:, None] * Bt
            o = (Ct * h).sum(-1)
            out.append(o if skip is None else o + skip * x[i, t])
        y = torch.stack(out) if out else x.new_zeros(0, D)
        if gate is not None:
            y = y * silu(gate[i, :count])
        rows.append(torch.cat((y, x.new_zeros(n - count, D))))
        states.append(h)
    return torch.stack(rows) if rows else x.new_zeros(x.shape), torch.stack(states) if states else x.new_zeros(0, D, A.shape[1])


def causal_conv(x, weight, bias=None, activation=None, initial=None, lengths=None):
    """(y [B,N,D], state [B,W-1,D]) of x [B,N,D] and weight [D,W], all float64."""
    b, n, D = x.shape
    W = weight.shape[1]
    front = x.new_zeros(b, W - 1, D) if initial is None else initial
    rows, states = [], []
    for i in range(b):
        count = n if lengths is None else min(max(int(lengths[i]), 0), n)
        wide = torch.cat((front[i], x[i, :count]))
        p = sum(wide[j:j + count] * weight[:, j] for j in range(W))
        if bias is not None:
            p = p + bias
        rows.append(torch.cat((silu(p) if activation == "silu" else p, x.new_zeros(n - count, D))))
        states.append(wide[count:])
    return torch.stack(rows) if rows else x.new_zeros(x.shape), torch.stack(states) if states else x.new_zeros(0, W - 1, D)


def rms_norm(x, weight=None, residual=None, eps=1e-5):
    """(y, s), float64, of x and residual in their own types; s as it is stored."""
    s = x.double() if residual is None else (x.float() + residual.float()).to(residual.dtype).double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.double()), s


def rms_norm_backward(dy, s, weight=None, dsum=None, eps=1e-5):
    """(ds, dweight) from the rows s that were normalised."""
    s, g = s.double(), dy.double()
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    gw = g if weight is None else g * weight.double()
    ds = r * (gw - s * r * r * (gw * s).mean(-1, keepdim=True))
    if dsum is not None:
        ds = ds + dsum.double()
    lead = tuple(range(s.ndim - (1 if weight is None else weight.ndim)))
    return ds, (g * s * r).sum(lead)
