"""GPU tests of rotary_embed against float64 rotations.

Bound: the angle keeps 2^-32 of a turn, and as an fp32 fraction half a step of it (2^-25 turns, 2^-22.3 rad); sine and
cosine in fp32 are within 4 half steps for fp32 results and within 2^-20 absolute for 16-bit ones (the hardware's
instructions, measured below 2^-21); two products and a sum: 3 half steps.  All relative to magnitude (|a| + |b|).
"""

import pytest
import torch

from oracle import mixer_ref
from tests.mixer_cases import DTYPES, randn, within

pytestmark = pytest.mark.gpu


def slack(dtype):
    return 2.0 ** -22.3 + (8 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -20)


def terms(x, plan):
    """magnitude (|a| + |b|) of each element's pair; copied elements are exact."""
    n, a = plan.rotary_dim // 2, x.double().abs()
    t = torch.zeros_like(a)
    if plan.interleaved:
        s = a[..., 0:2 * n:2] + a[..., 1:2 * n:2]
        t[..., 0:2 * n:2], t[..., 1:2 * n:2] = s, s
    else:
        s = a[..., :n] + a[..., n:2 * n]
        t[..., :n], t[..., n:2 * n] = s, s
    return abs(plan.magnitude) * t


def check(pkg, device, q, k, pos, plan, grads=True, place=lambda t: t):
    dt = q.dtype
    leaves = [place(q.to(device)).requires_grad_(grads)]
    if k is not None:
        leaves.append(place(k.to(device)).requires_grad_(grads))
    got = pkg.rotary_embed(leaves[0], leaves[1] if k is not None else None, pos.to(device), plan)
    assert (got[1] is None) == (k is None)
    outs, inputs = [t for t in got if t is not None], [t for t in (q, k) if t is not None]
    f = plan.inverse_frequencies
    for x, y in zip(inputs, outs):
        assert y.dtype == dt and y.shape == x.shape and y.transpose(1, 2).is_contiguous()
        within(y, mixer_ref.rotary(x, pos, f, plan.interleaved, plan.magnitude), terms(x, plan), dt, slack(dt))
        assert torch.equal(y[..., plan.rotary_dim:].cpu(), x[..., plan.rotary_dim:])
    if grads:
        g = torch.Generator().manual_seed(1)
        ups = [randn(g, *x.shape, dtype=dt) for x in inputs]
        back = torch.autograd.grad(outs, leaves, [place(u.to(device)) for u in ups])
        for u, d in zip(ups, back):
            within(d, mixer_ref.rotary(u, pos, f, plan.interleaved, plan.magnitude, inverse=True), terms(u, plan), dt, slack(dt))


def make(B, H, Hkv, N, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (randn(g, B, N, H, D, dtype=dtype).transpose(1, 2),
            randn(g, B, N, Hkv, D, dtype=dtype).transpose(1, 2) if Hkv else None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rd", [(64, 64), (64, 32), (64, 16), (64, 2), (64, 22), (128, 128), (2, 2), (10, 6), (72, 48)])
def test_shapes(pkg, device, dtype, interleaved, D, rd):
    plan = pkg.rotary_plan(rd, interleaved=interleaved, device=device)
    q, k = make(2, 3, 1, 5, D, dtype, seed=D + rd)
    check(pkg, device, q, k, torch.tensor([0, 1, 2, 100, 4095]), plan)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(pkg, device, dtype, interleaved):
    """2^20, 2^31 and negative positions; each sequence at its own place; every scaling."""
    pos = torch.tensor([[0, 1 << 20, (1 << 20) + 1], [(1 << 31) - 5, -7, 1 << 31]])
    for kw in ({}, dict(scaling="linear", factor=8.0), dict(scaling="base", factor=8.0),
               dict(scaling="bands", factor=64.0, original_length=2048, magnitude=1.4)):
        plan = pkg.rotary_plan(64, interleaved=interleaved, device=device, **kw)
        q, k = make(2, 4, 2, 3, 64, dtype, seed=3)
        # float64 angles of 2^31 rad are themselves off by 2^-22 rad
        check(pkg, device, q, k, pos, plan)


def test_head_counts_and_row_counts(pkg, device):
    plan = pkg.rotary_plan(64, device=device)
    for B, H, Hkv, N in ((1, 1, 1, 1), (1, 7, 0, 3), (256, 8, 2, 1), (3, 12, 4, 333), (2, 40, 5, 1500)):
        q, k = make(B, H, Hkv, N, 64, torch.bfloat16, seed=N)
        check(pkg, device, q, k, torch.arange(N) + 17, plan)


def test_layouts_and_position_types(pkg, device):
    """Head-major memory, rows off alignment, strided positions and int32: the bits of the plain call."""
    for interleaved in (False, True):
        plan = pkg.rotary_plan(64, interleaved=interleaved, device=device)
        q, k = make(2, 4, 2, 50, 64, torch.bfloat16, seed=4)
        pos = torch.arange(50) * 3

        def shifted(t):
            base = torch.zeros(*t.shape[:-1], 67, device=t.device, dtype=t.dtype)[..., 1:65]
            return base.copy_(t.detach()).detach()

        for place in (lambda t: t.detach().contiguous(), shifted):
            check(pkg, device, q, k, pos, plan, place=place)
        qd, kd = q.to(device), k.to(device)
        want = pkg.rotary_embed(qd, kd, pos.to(device), plan)
        wide = torch.arange(100, device=device, dtype=torch.int32) * 3 // 2
        for p in (pos.to(device).int(), wide[::2], pos.to(device).expand(2, 50), pos.to(device).repeat(2, 1).int()):
            got = pkg.rotary_embed(qd, kd, p, plan)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_copied_elements_take_nothing_from_their_neighbours(pkg, device):
    """NaN and infinities behind the turned part stay where they are."""
    for interleaved in (False, True):
        for rd in (32, 6):
            plan = pkg.rotary_plan(rd, interleaved=interleaved, magnitude=2.0, device=device)
            x = torch.ones(1, 1, 3, 64)
            x[..., rd], x[..., rd + 2], x[..., 63] = float("nan"), float("inf"), float("-inf")
            y, _ = pkg.rotary_embed(x.to(device), None, torch.arange(3, device=device), plan)
            assert torch.equal(y.cpu()[..., rd:].nan_to_num(7.0), x[..., rd:].nan_to_num(7.0))
            assert bool(y[..., :rd].isfinite().all())


def test_gradient_of_one_output_and_empty(pkg, device):
    plan = pkg.rotary_plan(64, device=device)
    q, k = (t.to(device).requires_grad_(True) for t in make(2, 4, 2, 9, 64, torch.float32, seed=5))
    pos = torch.arange(9, device=device)
    qo, ko = pkg.rotary_embed(q, k, pos, plan)
    dq, dk = torch.autograd.grad(ko, (q, k), torch.ones_like(ko), allow_unused=True)
    assert dq is None or not bool(dq.any())
    within(dk, mixer_ref.rotary(torch.ones(2, 2, 9, 64), pos.cpu(), plan.inverse_frequencies, False, inverse=True),
           terms(torch.ones(2, 2, 9, 64), plan), torch.float32, slack(torch.float32))
    e, _ = pkg.rotary_embed(q[:, :, :0], None, pos[:0], plan)
    assert e.shape == (2, 4, 0, 64)
    # the rotation is linear: a difference of any step is its gradient
    way = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(device)
    up = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).to(device)
    (g,) = torch.autograd.grad(pkg.rotary_embed(q, None, pos, plan)[0], q, up)
    with torch.no_grad():
        a, b = ((pkg.rotary_embed(q + s * way, None, pos, plan)[0].double() * up.double()).sum() for s in (1, -1))
    size = float(((q.abs() + way.abs()).double().sum(-1) * up.abs().amax(-1).double() * 2).sum())
    assert abs(float((a - b) / 2 - (g.double() * way.double()).sum())) <= 3 * slack(torch.float32) * size
    graph_q = q.detach().clone().requires_grad_(True)
    u = up.clone().requires_grad_(True)
    (first,) = torch.autograd.grad(pkg.rotary_embed(graph_q, None, pos, plan)[0], graph_q, u, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), u)


def test_graph_and_compile(pkg, device):
    plan = pkg.rotary_plan(32, interleaved=True, device=device)
    q, k = (t.to(device) for t in make(2, 4, 2, 40, 64, torch.bfloat16, seed=6))
    pos = torch.arange(40, device=device) + 1000

    def step(q, k):
        a, b = pkg.rotary_embed(q, k, pos, plan)
        return (a.float() ** 3).sum() + (b.float() ** 3).sum()

    results = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_(True) for t in (q, k)]
        loss = fn(*leaves)
        loss.backward()
        results.append([loss.detach(), *(t.grad for t in leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    pkg.rotary_embed(q, k, pos, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = pkg.rotary_embed(q, k, pos, plan)
    for rep in range(3):
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, pkg.rotary_embed(q, k, pos, plan))), rep
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_near_quarter_turns(pkg, device, dtype, interleaved):
    """Sines and cosines that are nearly 0, of angles around every quarter turn: in fp32 as exact as around angle 0.

    Exact: the plan's integer turns, the nearest quarter taken off in integers.  Bound in fp32: 2^-32 of a turn is cut off,
    and relative to the value half a step for the angle, 4 for sine and cosine, 2 for the products; 16-bit results add the
    hardware's 2^-20 and their own rounding."""
    import math
    from fractions import Fraction
    g = torch.Generator().manual_seed(9)
    near = torch.tensor([q / 4 + s * d for q in range(-3, 5) for s in (1, -1) for d in (3.0e-7, 2.87e-6, 1.3e-4, 0.011, 0.1249)])
    f = 2 * math.pi * (near.double() + 1e-9 * torch.rand(near.numel(), generator=g, dtype=torch.float64))
    plan = pkg.rotary_plan(2 * f.numel(), inverse_frequencies=f, interleaved=interleaved, device=device)
    n = f.numel()
    x = torch.zeros(1, 1, 3, 2 * n)
    (x[..., 0::2] if interleaved else x[..., :n]).fill_(1.0)   # pairs (1, 0): the results are the cosine and the sine
    positions = torch.tensor([0, 1, 1023])
    y = pkg.rotary_embed(x.to(device=device, dtype=dtype), None, positions.to(device), plan)[0].cpu().double()
    c, s = (y[0, 0, :, 0::2], y[0, 0, :, 1::2]) if interleaved else (y[0, 0, :, :n], y[0, 0, :, n:])
    step = {torch.float32: 8 * 2.0 ** -24, torch.bfloat16: 2.0 ** -8 + 8 * 2.0 ** -24, torch.float16: 2.0 ** -11 + 8 * 2.0 ** -24}[dtype]
    floor = 2 * math.pi * 2.0 ** -32 + (0 if dtype == torch.float32 else 2.0 ** -20 + (2.0 ** -25 if dtype == torch.float16 else 0))
    for i, p in enumerate(positions.tolist()):
        for j, t in enumerate(plan.turns.tolist()):
            at = Fraction(p * t % 2 ** 64, 2 ** 64)
            quarter = round(4 * at)
            rest = float(at - Fraction(quarter, 4)) * 2 * math.pi
            sn, cs = math.sin(rest), math.cos(rest)
            for _ in range(quarter % 4):
                sn, cs = cs, -sn
            for got, want in ((float(s[i, j]), sn), (float(c[i, j]), cs)):
                assert abs(got - want) <= floor + step * abs(want), (p, float(at), got, want)
