"""The selective mixer's oracle against other statements of the same definitions: sums over pairs of tokens, torch's
convolution, differences."""

import math

import torch

from oracle import selective_ref as ref


def make_scan(seed, b=2, n=9, D=6, S=5, G=2):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)   # noqa: E731
    return dict(x=r(b, n, D), delta=r(b, n, D), A=-r(D, S).exp(), B=r(b, n, G, S), C=r(b, n, G, S), skip=r(D), gate=r(b, n, D),
                delta_bias=r(D), initial=r(b, D, S))


def test_scan_is_the_sum_over_pairs_of_tokens():
    """y_t = sum_{j <= t} C_t . exp(A sum_{j < i <= t} step_i) step_j x_j B_j, plus the initial state's share."""
    a = make_scan(1)
    b, n, D = a["x"].shape
    step = torch.nn.functional.softplus(a["delta"] + a["delta_bias"])
    y, state = ref.selective_scan(**a, softplus=True)
    per = D // a["B"].shape[2]
    B, C = (a[k].repeat_interleave(per, 2) for k in ("B", "C"))
    for i in range(b):
        cum = step[i].cumsum(0)
        for t in range(n):
            h = torch.exp(cum[t][:, None] * a["A"]) * a["initial"][i]
            for j in range(t + 1):
                h = h + torch.exp((cum[t] - cum[j])[:, None] * a["A"]) * (step[i, j] * a["x"][i, j])[:, None] * B[i, j]
            o = ((h * C[i, t]).sum(-1) + a["skip"] * a["x"][i, t]) * torch.nn.functional.silu(a["gate"][i, t])
            assert torch.allclose(o, y[i, t], rtol=1e-12, atol=1e-12)
        assert torch.allclose(h, state[i], rtol=1e-12, atol=1e-12)


def test_scan_lengths_and_parts():
    """A shortened sequence is the sequence cut off, and two parts with the state between them are the whole."""
    a = make_scan(2, n=12)
    lengths = torch.tensor([5, 0])
    y, state = ref.selective_scan(**a, lengths=lengths)
    cut = {k: v[:1, :5] if k in ("x", "delta", "B", "C", "gate") else v[:1] if k == "initial" else v for k, v in a.items()}
    y0, s0 = ref.selective_scan(**cut)
    assert torch.equal(y[0, :5], y0[0]) and not y[0, 5:].any() and not y[1].any()
    assert torch.equal(state[0], s0[0]) and torch.equal(state[1], a["initial"][1])
    whole, end = ref.selective_scan(**a)
    one = {k: v[:, :7] if k in ("x", "delta", "B", "C", "gate") else v for k, v in a.items()}
    two = {k: v[:, 7:] if k in ("x", "delta", "B", "C", "gate") else v for k, v in a.items()}
    ya, mid = ref.selective_scan(**one)
    two["initial"] = mid
    yb, last = ref.selective_scan(**two)
    assert torch.equal(torch.cat((ya, yb), 1), whole) and torch.equal(last, end)


def test_scan_gradients_by_differences():
    a = make_scan(3, b=1, n=4, D=2, S=2, G=1)
    names = list(a)
    leaves = [a[k].clone().requires_grad_(True) for k in names]
    f = lambda *t: ref.selective_scan(**dict(zip(names, t)), softplus=True)   # noqa: E731
    assert torch.autograd.gradcheck(f, leaves)


def test_softplus_of_any_step():
    """log(1 + e^x) and its slope 1 / (1 + e^-x), at 0 and far away too."""
    x = torch.tensor([0.0, -0.0, 1e-9, 3.0, -3.0, 40.0, -40.0, -800.0, 800.0, -float("inf")], dtype=torch.float64, requires_grad=True)
    one = torch.ones(1, 1, 1, dtype=torch.float64)
    y, _ = ref.selective_scan(one.expand(1, 1, 10), x.view(1, 1, 10), -one[0].expand(10, 1), one, one, softplus=True)
    slope, = torch.autograd.grad(y.sum(), x)
    want = [math.log1p(math.exp(min(v, 30.0))) if v < 30 else v for v in x.tolist()]
    assert torch.allclose(y[0, 0], torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)
    assert torch.allclose(slope, 1 / (1 + torch.exp(-x.detach())), rtol=1e-13, atol=0)


def test_conv_is_torchs_convolution():
    g = torch.Generator().manual_seed(4)
    x, w, c = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 11, 5), (5, 4), (5,)))
    front = torch.randn(2, 3, 5, generator=g, dtype=torch.float64)
    y, state = ref.causal_conv(x, w, c, None, front)
    want = torch.nn.functional.conv1d(torch.cat((front, x), 1).transpose(1, 2), w[:, None], c, groups=5).transpose(1, 2)
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12) and torch.equal(state, x[:, -3:])
    y, state = ref.causal_conv(x, w, c, "silu", front, torch.tensor([2, 0]))
    assert torch.allclose(y[0, :2], torch.nn.functional.silu(want[0, :2]), rtol=1e-12) and not y[0, 2:].any() and not y[1].any()
    assert torch.equal(state[0], torch.cat((front[0, 2:], x[0, :2]))) and torch.equal(state[1], front[1])


def test_rms_norm_and_its_gradients():
    g = torch.Generator().manual_seed(5)
    x, w, dy, ds = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 2, 7), (2, 7), (3, 2, 7), (3, 2, 7)))
    y, s = ref.rms_norm(x, w)
    assert torch.allclose(y, torch.nn.functional.rms_norm(x, (7,), eps=1e-5) * w, rtol=1e-12)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    yl = xl / torch.sqrt((xl * xl).mean(-1, keepdim=True) + 1e-5) * wl
    dx, dw = torch.autograd.grad((yl * dy).sum() + (xl * ds).sum(), (xl, wl))
    got = ref.rms_norm_backward(dy, s, w, ds)
    assert torch.allclose(got[0], dx, rtol=1e-12, atol=1e-12) and torch.allclose(got[1], dw, rtol=1e-12, atol=1e-12)
    lo = torch.randn(4, 9, generator=g).bfloat16()
    _, s = ref.rms_norm(lo, residual=lo)
    assert torch.equal(s, (lo.float() * 2).bfloat16().double())
