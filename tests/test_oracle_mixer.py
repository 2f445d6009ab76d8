"""The mixer's oracle (oracle/mixer_ref.py) against autograd, differences and closed forms (CPU)."""

import math

import pytest
import torch

from oracle import mixer_ref


def inputs(B=2, H=4, Hkv=2, N=9, D=6, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)   # noqa: E731
    return (r(B, H, N, D), r(B, Hkv, N, D), r(B, Hkv, N, D), -torch.rand(H, generator=g, dtype=torch.float64),
            r(B, H, D, D), r(B, H, N, D), r(B, H, D, D))


def quadratic(q, k, v, lg, scale, S0, lengths):
    """The same as one masked sum over pairs, for autograd."""
    B, H, N, D = q.shape
    k, v = (x.repeat_interleave(H // k.shape[1], 1) for x in (k, v))
    t = torch.arange(N)
    live = (t[None] < lengths[:, None])[:, None, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    gap = (t[:, None] - t[None]).clamp(min=0)
    w = torch.where(t[:, None] >= t[None], torch.exp(lg[:, None, None] * gap), 0.0)
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * w, v) + torch.exp(lg[:, None] * (t + 1))[..., None] * torch.matmul(q, S0)
    until = (lengths[:, None] - 1 - t).clamp(min=0)
    kw = k * torch.exp(lg[None, :, None] * until[:, None])[..., None]
    state = torch.exp(lg[None, :] * lengths[:, None])[..., None, None] * S0 + torch.matmul(kw.transpose(-1, -2), v)
    return torch.where(live, scale * o, 0.0), state


def test_recurrence_equals_the_sum_over_pairs_and_its_gradients():
    q, k, v, lg, S0, do, dS = inputs()
    lengths = torch.tensor([9, 5])
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, lg, S0)]
    o, s = quadratic(*leaves[:4], 0.3, leaves[4], lengths)
    out, state = mixer_ref.linear_attention(q, k, v, lg, 0.3, S0, lengths)
    torch.testing.assert_close(out, o.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(state, s.detach(), rtol=1e-12, atol=1e-12)
    want = torch.autograd.grad((o, s), leaves, (do, dS))
    dq, dk, dv, dlg, dS0 = mixer_ref.linear_attention_backward(q, k, v, lg, 0.3, do, S0, lengths, dS)
    for a, b in zip((dq, dk, dv, dlg, dS0), want):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)


def test_decay_edges():
    """A decay of 0 keeps the token alone, of 1 sums everything, and values above 0 count as 0."""
    q, k, v, _, _, do, _ = inputs(H=2, Hkv=2)
    lg = torch.tensor([-math.inf, 0.0], dtype=torch.float64)
    out, _ = mixer_ref.linear_attention(q, k, v, lg, 1.0)
    alone = (q[:, 0] * k[:, 0]).sum(-1, keepdim=True) * v[:, 0]
    torch.testing.assert_close(out[:, 0], alone)
    running = torch.cumsum(k[:, 1, :, :, None] * v[:, 1, :, None, :], 1)
    torch.testing.assert_close(out[:, 1], torch.einsum("bnd,bnde->bne", q[:, 1], running))
    above, _ = mixer_ref.linear_attention(q, k, v, torch.tensor([-math.inf, 0.7], dtype=torch.float64), 1.0)
    assert torch.equal(above, out)
    assert mixer_ref.linear_attention_backward(q, k, v, torch.tensor([-0.1, 0.7]), 1.0, do)[3][1] == 0


def test_rotary_is_a_rotation_and_its_inverse_undoes_it():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, 10, generator=g, dtype=torch.float64)
    pos = torch.tensor([0, 1, 7, 1000, 1 << 20])
    f = torch.tensor([1.0, 0.3, 0.01], dtype=torch.float64)
    for interleaved in (False, True):
        y = mixer_ref.rotary(x, pos, f, interleaved)
        assert torch.equal(y[..., 6:], x[..., 6:]) and torch.equal(y[:, :, 0], x[:, :, 0])
        torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
        torch.testing.assert_close(mixer_ref.rotary(y, pos, f, interleaved, inverse=True), x)
        a = 7 * 0.3   # pair 1 of position 7
        i, j = (2, 3) if interleaved else (1, 4)
        want = x[0, 0, 2, i] * math.cos(a) - x[0, 0, 2, j] * math.sin(a)
        assert abs(float(y[0, 0, 2, i] - want)) < 1e-12


def test_layer_norm_gradients_match_autograd():
    g = torch.Generator().manual_seed(2)
    for shape in ((5, 7), (3, 4, 6)):
        x = torch.randn(*shape, generator=g, dtype=torch.float64, requires_grad=True)
        w, b = (torch.randn(*shape[1:], generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
        dy = torch.randn(*shape, generator=g, dtype=torch.float64)
        y = torch.nn.functional.layer_norm(x, shape[-1:], eps=1e-3) * w + b
        torch.testing.assert_close(mixer_ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-3), y.detach())
        for a, want in zip(mixer_ref.layer_norm_backward(dy, x.detach(), w.detach(), 1e-3),
                           torch.autograd.grad(y, (x, w, b), dy)):
            torch.testing.assert_close(a, want)


@pytest.mark.parametrize("lengths,state", [(None, True), ([150, 64, 0], True), ([65, 1, 149], False)])
def test_chunked_attention_is_the_recurrence(lengths, state):
    """Outputs, states and gradients in blocks of tokens, and the terms that cross a block's border."""
    g = torch.Generator().manual_seed(5)
    B, H, Hkv, N, D = 3, 4, 2, 150, 8
    q, dout = (torch.randn(B, H, N, D, generator=g) for _ in range(2))
    k, v = (torch.randn(B, Hkv, N, D, generator=g) for _ in range(2))
    lg = torch.tensor([-0.5, -0.01, 0.0, 0.3])
    S0, dS = (torch.randn(B, H, D, D, generator=g) for _ in range(2))
    dS = dS if state else None
    out, end, grads, crossing = mixer_ref.linear_attention_chunked(q, k, v, lg, 0.3, dout, S0, lengths, dS)
    want = mixer_ref.linear_attention(q, k, v, lg, 0.3, S0, lengths)
    wgrads = mixer_ref.linear_attention_backward(q, k, v, lg, 0.3, dout, S0, lengths, dS)
    for a, b in zip((out, end, *grads), (*want, *wgrads)):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)
    for b in range(B):
        n = N if lengths is None else lengths[b]
        assert len(crossing[b]) == -(-n // 64)
        if n:   # what enters times its adjoint
            torch.testing.assert_close(crossing[b][0], (S0[b].double() * grads[4][b]).sum((1, 2)), rtol=1e-11, atol=1e-11)
