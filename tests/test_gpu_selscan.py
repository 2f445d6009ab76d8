"""GPU tests of selective_scan and selective_scan_step against the float64 recurrence, with selective_cases' bounds: what
each rounding of the recurrence can do, carried along it."""

import pytest
import torch

from oracle import selective_ref
from tests.mixer_cases import DTYPES, randn
from tests.selective_cases import U, f64, scan_bounds, segment_tokens, within

pytestmark = pytest.mark.gpu
ALL = ("skip", "gate", "delta_bias", "initial")


def case(device, B, N, D, S, dtype, G=None, parts=ALL, softplus=True, lengths=None, seed=0, atype=torch.float32, index=torch.int32):
    g = torch.Generator().manual_seed(seed)
    rows = (B, N, S) if G is None else (B, N, G, S)
    c = dict(x=randn(g, B, N, D, dtype=dtype),
             delta=(randn(g, B, N, D) if softplus else 0.4 * torch.rand(B, N, D, generator=g)).to(dtype),
             A=-torch.exp(0.5 * randn(g, D, S)).to(atype), B=randn(g, *rows, dtype=dtype), C=randn(g, *rows, dtype=dtype))
    more = dict(skip=randn(g, D, dtype=atype), gate=randn(g, B, N, D, dtype=dtype),
                delta_bias=(randn(g, D) if softplus else 0.1 * torch.rand(D, generator=g)).to(atype), initial=randn(g, B, D, S))
    c.update({k: v for k, v in more.items() if k in parts})
    c = {k: v.to(device).requires_grad_(True) for k, v in c.items()}
    c["softplus"], c["lengths"] = softplus, None if lengths is None else torch.tensor(lengths, dtype=index, device=device)
    c["dy"], c["dstate"] = randn(g, B, N, D, dtype=dtype).to(device), randn(g, B, D, S).to(device)
    return c


def leaves_of(c):
    return [k for k in ("x", "delta", "A", "B", "C", *ALL) if k in c]


def call(pkg, c, return_state=True):
    return pkg.selective_scan(c["x"], c["delta"], c["A"], c["B"], c["C"], skip=c.get("skip"), gate=c.get("gate"),
                              delta_bias=c.get("delta_bias"), softplus=c["softplus"], initial_state=c.get("initial"),
                              lengths=c["lengths"], return_state=return_state)


def check(pkg, c, use=("y", "state")):
    out = dict(zip(("y", "state"), call(pkg, c)))
    names, ups = leaves_of(c), dict(y=c["dy"], state=c["dstate"])
    grads = torch.autograd.grad([out[o] for o in use], [c[k] for k in names], [ups[o] for o in use])
    lengths = None if c["lengths"] is None else c["lengths"].cpu()
    ref = {k: f64(c[k]).requires_grad_(True) for k in names}
    want = dict(zip(("y", "state"), selective_ref.selective_scan(**ref, softplus=c["softplus"], lengths=lengths)))
    wants = torch.autograd.grad([want[o] for o in use], list(ref.values()), [f64(ups[o]) for o in use], allow_unused=True)
    dy = f64(c["dy"]) if "y" in use else torch.zeros_like(f64(c["dy"]))
    off = scan_bounds({k: v.detach() for k, v in ref.items()}, c["softplus"], lengths, dy, f64(c["dstate"]) if "state" in use else None)
    dtype = c["x"].dtype
    within(out["y"], want["y"].detach(), off["y"], dtype, U)
    within(out["state"], want["state"].detach(), off["state"], torch.float32, U)
    for k, g, w in zip(names, grads, wants):
        assert g.dtype == c[k].dtype and g.shape == c[k].shape
        within(g, torch.zeros_like(off[k]) if w is None else w, off[k], c[k].dtype, U)
    if lengths is not None:
        dead = torch.arange(c["x"].shape[1])[None] >= lengths[:, None]
        for k, t in (("y", out["y"]), *((k, g) for k, g in zip(names, grads) if k in ("x", "delta", "gate", "B", "C"))):
            assert not bool(t.detach().cpu()[dead].any()), k
    return out, dict(zip(names, grads))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("S", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64])
def test_states(pkg, device, S, dtype):
    """Every way states are shared by lanes, filled or not, rows taken in vectors and by elements."""
    check(pkg, case(device, 2, 37, 40, S, dtype, seed=S))
    check(pkg, case(device, 1, 41, 13, S, dtype, seed=S))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 129, 200])
@pytest.mark.parametrize("S", [4, 16, 24, 40])
def test_token_counts(pkg, device, N, S, dtype):
    """Around the tiles', chunks' and segments' ends."""
    assert (N > 64) == segment_tokens(1, N, 24, 1, S)[1]
    check(pkg, case(device, 1, N, 24, S, dtype, seed=N))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [1, 2, 3, 4, 7, 8, 9, 16, 63, 64, 65, 72, 200])
def test_channel_counts(pkg, device, D, dtype):
    check(pkg, case(device, 2, 70, D, 16, dtype, seed=D))


@pytest.mark.parametrize("dtype", DTYPES[::2], ids=str)
@pytest.mark.parametrize("G,D", [(1, 40), (2, 144), (3, 192), (5, 40), (5, 35), (12, 12), (4, 288)])
@pytest.mark.parametrize("S", [5, 16, 32, 64])
def test_groups(pkg, device, G, D, S, dtype):
    """Channels that share B and C: groups of whole workgroups, parts of one, single channels."""
    check(pkg, case(device, 2, 45, D, S, dtype, G=G, seed=G))


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("parts", [(), ("skip",), ("gate",), ("delta_bias",), ("initial",), ("skip", "gate"), ALL], ids=str)
def test_parts(pkg, device, parts, softplus):
    for use in (("y",), ("state",), ("y", "state")):
        check(pkg, case(device, 2, 75, 24, 16, torch.bfloat16, parts=parts, softplus=softplus), use)
    check(pkg, case(device, 2, 75, 21, 6, torch.float32, parts=parts, softplus=softplus))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_table_types(pkg, device, dtype):
    check(pkg, case(device, 2, 20, 16, 8, torch.bfloat16, atype=dtype))


@pytest.mark.parametrize("S", [4, 16, 64])
@pytest.mark.parametrize("B,N,D", [(200, 70, 8), (50, 100, 260), (1, 1500, 8), (3, 300, 64)])
def test_one_segment_and_many(pkg, device, B, N, D, S):
    """Enough channels for one segment, and sequences cut into as many as are joined."""
    check(pkg, case(device, B, N, D, S, torch.float32, seed=N))


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=str)
@pytest.mark.parametrize("S,parts", [(16, ALL), (8, ALL), (13, ("skip",))])
def test_tiles_of_long_segments(pkg, device, S, parts, dtype):
    """Rows of 16 bits in one segment of several tiles (64 tokens forward up to 16 states), the last one not whole; sequences
    that end in the first, second and third tile."""
    assert not segment_tokens(4, 150, 3080, 1, S)[1]
    check(pkg, case(device, 4, 150, 3080, S, dtype, parts=parts, lengths=[150, 65, 64, 129], seed=S))
    check(pkg, case(device, 4, 70, 3080, S, dtype, parts=parts, seed=S + 1))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [65, 127, 128, 129, 200])
@pytest.mark.parametrize("S,parts", [(8, ALL), (16, ALL), (16, ("skip", "initial")), (24, ALL)])
def test_one_call_is_its_parts_of_one_tile(pkg, device, S, parts, N, dtype):
    """A segment of several tiles against calls of 64 tokens with the state and its gradient between them: the same bits of
    everything but the sums over all tokens."""
    B, D = 22, 520
    assert not segment_tokens(B, N, D, 1, S)[1]
    ends = [N, N - 1, 64, 65, 63, 1, 0, 128, 129]
    c = case(device, B, N, D, S, dtype, parts=parts, lengths=[min(ends[i % len(ends)], N) for i in range(B)], seed=N)
    rows = [k for k in ("x", "delta", "B", "C", "gate") if k in c]
    out = call(pkg, c)
    grads = dict(zip([*rows, "initial"], torch.autograd.grad(out, [c[k] for k in [*rows, "initial"]], [c["dy"], c["dstate"]])))
    calls, state = [], c["initial"]
    for a in range(0, N, 64):
        d = dict(c, **{k: c[k].detach()[:, a:a + 64].contiguous().requires_grad_(True) for k in rows},
                 initial=state.detach().requires_grad_(True), lengths=(c["lengths"] - a).clamp(min=0))
        y, state = call(pkg, d)
        calls.append((a, d, y, state))
    same([torch.cat([y for _, _, y, _ in calls], 1), state], out)
    dstate, parts_of = c["dstate"], {k: [] for k in rows}
    for a, d, y, s in reversed(calls):
        *g, dstate = torch.autograd.grad([y, s], [d[k] for k in [*rows, "initial"]], [c["dy"][:, a:a + 64].contiguous(), dstate])
        for k, t in zip(rows, g):
            parts_of[k].insert(0, t)
    same([*(torch.cat(parts_of[k], 1) for k in rows), dstate], [grads[k] for k in [*rows, "initial"]])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,S,parts", [(24, 16, ALL), (13, 5, ALL), (16, 40, ("gate",)), (24, 16, ())])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_lengths(pkg, device, D, S, parts, index, dtype):
    """Sequences that end inside tiles, chunks and segments, at their ends, nowhere, before the first token."""
    lengths = [150, 0, 1, 64, 65, 31, -4, 999, 128, 97]
    check(pkg, case(device, 10, 150, D, S, dtype, parts=parts, lengths=lengths, index=index))


def test_values_behind_the_lengths_are_not_used(pkg, device):
    """NaN and infinities behind the end, in rows and their gradients: the bits of zeros there."""
    for D, S in ((24, 16), (13, 5)):
        c = case(device, 4, 140, D, S, torch.bfloat16, lengths=[70, 0, 33, 129])
        dead = torch.arange(140, device=device)[None] >= c["lengths"][:, None]
        results = []
        for fill in (0.0, float("nan"), float("inf"), -float("inf")):
            d = dict(c)
            for k in ("x", "delta", "gate", "B", "C", "dy"):
                d[k] = c[k].detach().masked_fill(dead[..., None], fill).requires_grad_(k != "dy")
            out = call(pkg, d)
            results.append([*out, *torch.autograd.grad(out, [d[k] for k in leaves_of(d)], [d["dy"], c["dstate"]])])
        for other in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(other, results[0]))


@pytest.mark.parametrize("S,D", [(16, 24), (5, 13), (64, 8)])
@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.bfloat16).min])
def test_steps_masked_by_delta(pkg, device, S, D, low):
    """A delta of minus infinity, or the type's lowest value, makes a step of 0: the state passes, and the other tokens'
    results are those of the sequence without the masked ones."""
    c = case(device, 2, 50, D, S, torch.bfloat16)
    keep = torch.arange(50, device=device) % 3 != 1
    d = dict(c, delta=c["delta"].detach().masked_fill(~keep[None, :, None], low).requires_grad_(True))
    out = call(pkg, d)
    grads = dict(zip(leaves_of(d), torch.autograd.grad(out, [d[k] for k in leaves_of(d)], [c["dy"], c["dstate"]])))
    e = dict(c, **{k: c[k].detach()[:, keep].requires_grad_(True) for k in ("x", "delta", "B", "C", "gate")})
    want = call(pkg, e)
    assert torch.equal(out[0][:, keep], want[0]) and torch.equal(out[1], want[1])
    assert all(bool(g.isfinite().all()) for g in grads.values()) and not bool(grads["delta"][:, ~keep].any())
    d["dy"] = c["dy"] * keep[None, :, None]
    part = torch.autograd.grad(call(pkg, d), [d["delta"], d["x"]], [d["dy"], c["dstate"]])
    part2 = torch.autograd.grad(want, [e["delta"], e["x"]], [c["dy"][:, keep], c["dstate"]])
    assert all(torch.equal(a[:, keep], b) for a, b in zip(part, part2))


def test_states_that_do_not_last(pkg, device):
    """A of minus infinity: nothing is kept from token to token, the results and gradients are finite."""
    c = case(device, 2, 100, 16, 8, torch.float32, parts=("initial",))
    for S in (0, 5):
        A = [c["A"].detach().clone() for _ in range(2)]
        A[0][:, S], A[1][:, S] = -float("inf"), -1e30
        results = []
        for a in A:
            d = dict(c, A=a.requires_grad_(True))
            out = call(pkg, d)
            results.append([*out, *torch.autograd.grad(out, [d[k] for k in leaves_of(d)], [c["dy"], c["dstate"]])])
        assert all(torch.equal(s, t) and bool(s.isfinite().all()) for s, t in zip(*results))


@pytest.mark.parametrize("S,D", [(8, 16), (16, 24), (5, 13), (40, 8)])
@pytest.mark.parametrize("softplus", [False, True])
def test_gradients_of_states_that_do_not_last(pkg, device, softplus, S, D):
    """A of minus infinity beside every input, sequences that end inside a chunk, steps of 0 and large gradients of the state:
    m = dstate h of a token whose step is 0 times a rate of -3.4e38 is out of range, and the token's part in the gradients of
    its step and of the bias is still 0.  All are finite and those of a rate of -1e30."""
    c = case(device, 4, 100, D, S, torch.float32, softplus=softplus, lengths=[100, 37, 64, 0])
    c["dstate"] = 1e3 * c["dstate"]
    if softplus:   # a step of 0; without the softplus only tokens behind the end have one
        masked = torch.arange(100, device=device) % 7 == 3
        c["delta"] = c["delta"].detach().masked_fill(masked[None, :, None], -float("inf")).requires_grad_(True)
    results = []
    for low in (-float("inf"), -1e30):
        A = c["A"].detach().clone()
        A[:, S // 2] = low
        d = dict(c, A=A.requires_grad_(True))
        out = call(pkg, d)
        results.append([*out, *torch.autograd.grad(out, [d[k] for k in leaves_of(d)], [c["dy"], c["dstate"]])])
    for k, s, t in zip(("y", "state", *leaves_of(c)), *results):
        assert bool(s.isfinite().all()) and torch.equal(s, t), k


@pytest.mark.parametrize("softplus", [False, True])
def test_steps_that_are_not_numbers_show_in_every_gradient(pkg, device, softplus):
    """A NaN among the steps reaches the outputs behind it and its channel's gradients; other channels' rows are untouched."""
    c = case(device, 1, 60, 24, 16, torch.float32, softplus=softplus)
    bad = c["delta"].detach().clone()
    bad[0, 40, 5] = float("nan")
    got = call(pkg, dict(c, delta=bad))
    d = dict(c, delta=bad.requires_grad_(True))
    names = ("x", "delta", "A", "delta_bias", "initial")
    grads = dict(zip(names, torch.autograd.grad(call(pkg, d), [d[k] for k in names], [c["dy"], c["dstate"]])))
    assert bool(got[0][0, 40:, 5].isnan().all()) and bool(got[0][0, :40].isfinite().all()) and bool(got[0][0, :, 6:].isfinite().all())
    assert bool(grads["x"][0, :41, 5].isnan().all()) and bool(grads["delta"][0, :41, 5].isnan().all())
    assert bool(grads["A"][5].isnan().all()) and bool(grads["delta_bias"][5].isnan()) and bool(grads["initial"][0, 5].isnan().all())
    other = torch.arange(24, device=device) != 5
    assert all(bool(grads[k][..., other].isfinite().all()) for k in ("x", "delta", "delta_bias"))


def test_growing_states_after_a_start_of_zeros(pkg, device):
    """A above 0 whose growth over a segment is beyond fp32: where nothing has entered yet nothing is multiplied."""
    c = case(device, 1, 200, 8, 4, torch.float32, parts=(), softplus=False)
    with torch.no_grad():
        c["A"].fill_(30.0)
        c["delta"].fill_(0.2)
        c["x"][:, :190] = 0
        y, state = call(pkg, c)
    assert segment_tokens(1, 200, 8, 1, 4)[1] and not bool(y[:, :190].any()) and bool(y.isfinite().all()) and bool(state.isfinite().all())


def test_steps_of_any_size(pkg, device):
    """delta from far below to far above: softplus against float64, through a scan of one token."""
    raw = torch.cat((torch.linspace(-30, 30, 4001), torch.tensor([-87.0, -100.0, -1e4, 1e4, 60.0])))
    D = raw.numel()
    one = torch.ones(1, 1, 1)
    y = pkg.selective_scan(torch.ones(1, 1, D, device=device), raw.view(1, 1, D).to(device), -torch.ones(D, 1, device=device),
                           one.to(device), one.to(device), softplus=True)[0, 0].double().cpu()
    want = torch.log1p(torch.exp(-raw.double().abs())) + raw.double().clamp(min=0)
    assert bool(((y - want).abs() <= want * 8 * U + 1.2e-38).all())


def same(a, b):
    assert len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


def test_layouts_give_the_same_bits(pkg, device):
    """Strided, expanded, misaligned inputs and gradients against contiguous ones."""
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t)   # noqa: E731
    apart = lambda t: torch.stack((t, t), -1)[..., 0]                                                     # noqa: E731
    wide = lambda t: torch.cat((t, t, t), -1)[..., t.shape[-1]:2 * t.shape[-1]]                            # noqa: E731
    turned = lambda t: t if t.ndim < 2 else t.transpose(0, 1).contiguous().transpose(0, 1)                # noqa: E731
    for dtype in DTYPES:
        for D, S, G in ((32, 16, 2), (32, 5, None), (12, 8, 3)):
            c = case(device, 3, 77, D, S, dtype, G=G, lengths=[77, 40, 0])

            def results(change):
                d = {k: change(v.detach()).requires_grad_(True) if k in leaves_of(c) else v for k, v in c.items()}
                out = call(pkg, d)
                return [*out, *torch.autograd.grad(out, [d[k] for k in leaves_of(c)], [change(c["dy"]), change(c["dstate"])])]

            want = results(lambda t: t)
            for change in (odd, apart, wide, turned):
                same(results(change), want)
    c = case(device, 3, 77, 32, 16, torch.bfloat16, parts=("gate",))
    d = dict(c, **{k: c[k].detach()[:1, :1].expand_as(c[k]) for k in ("x", "delta", "gate", "B", "C")})
    e = dict(d, **{k: d[k].contiguous() for k in ("x", "delta", "gate", "B", "C")})
    same(call(pkg, d), call(pkg, e))
    x = c["x"].detach()[:1, :1].clone().requires_grad_(True)   # the gradient of a broadcast input is the sum
    f = dict(c, x=x.expand(3, 77, 32))
    g = dict(c, x=x.expand(3, 77, 32).detach().clone().requires_grad_(True))
    dx, = torch.autograd.grad(call(pkg, f), x, [c["dy"], c["dstate"]])
    dw, = torch.autograd.grad(call(pkg, g), g["x"], [c["dy"], c["dstate"]])
    assert torch.equal(dx, dw.sum((0, 1), keepdim=True))


def test_tokens_far_apart(pkg, device):
    """Token strides of 2^22 elements and more, sequences past 2^31, one token with a stride of its own."""
    c = case(device, 2, 40, 24, 16, torch.bfloat16, parts=("gate",))
    buf = torch.empty((1 << 31) + (1 << 28), dtype=torch.bfloat16, device=device)
    with torch.no_grad():
        want = call(pkg, c)
        for token in ((1 << 22) - 8, 1 << 22, (1 << 22) + 5):
            far = buf.as_strided((2, 40, 24), ((1 << 31) - 8, token, 1)) if token < 1 << 22 else buf.as_strided((2, 40, 24), (41 * token, token, 1))
            same(call(pkg, dict(c, x=far.copy_(c["x"]))), want)
            rows = buf.as_strided((2, 40, 16), far.stride())
            same(call(pkg, dict(c, B=rows.copy_(c["B"]))), want)
        one = dict(c, **{k: c[k][:, :1] for k in ("x", "delta", "gate", "B", "C")})
        same(call(pkg, dict(one, x=buf.as_strided((2, 1, 24), (1 << 23, 1 << 25, 1)).copy_(one["x"]))), call(pkg, one))


def test_differences(pkg, device):
    """Every gradient against central differences of the float64 recurrence."""
    c = case(device, 1, 70, 5, 3, torch.float32)
    out = call(pkg, c)
    names = leaves_of(c)
    grads = torch.autograd.grad(out, [c[k] for k in names], [c["dy"], c["dstate"]])

    def f(v):
        y, s = selective_ref.selective_scan(**v, softplus=True)
        return float((y * f64(c["dy"])).sum() + (s * f64(c["dstate"])).sum())

    h, at = 1e-5, {k: f64(c[k]) for k in names}
    for k, grad in zip(names, grads):
        for i in range(0, grad.numel(), max(grad.numel() // 5, 1)):
            d = []
            for sign in (1, -1):
                v = dict(at, **{k: at[k].clone()})
                v[k].view(-1)[i] += sign * h
                d.append(f(v))
            # the difference: 1e-13 / h of rounding and h^2 of third derivatives; the gradient's own bound is tested above
            assert abs((d[0] - d[1]) / (2 * h) - float(grad.reshape(-1)[i])) < 1e-3 * (1 + abs(float(grad.reshape(-1)[i]))), (k, i)


def test_empty(pkg, device):
    c = case(device, 2, 0, 16, 8, torch.bfloat16)
    y, s = call(pkg, c)
    assert y.shape == (2, 0, 16) and torch.equal(s, c["initial"])
    grads = torch.autograd.grad([y, s], [c[k] for k in leaves_of(c)], [c["dy"], c["dstate"]])
    assert torch.equal(grads[-1], c["dstate"]) and not any(bool(g.any()) for g in grads[:-1])
    c = case(device, 0, 7, 16, 8, torch.bfloat16)
    out = call(pkg, c)
    grads = torch.autograd.grad(out, [c[k] for k in leaves_of(c)], [c["dy"], c["dstate"]])
    assert out[0].shape == (0, 7, 16) and out[1].shape == (0, 16, 8) and not any(bool(g.any()) for g in grads)


def test_refusals(pkg, device):
    import torch.autograd.forward_ad as fw
    c = case(device, 1, 9, 16, 8, torch.float32, parts=())
    g, = torch.autograd.grad(call(pkg, c, False).sum(), c["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        g.sum().backward()
    for k in leaves_of(c):
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            call(pkg, dict(c, **{k: fw.make_dual(c[k].detach(), torch.ones_like(c[k]))}))
    with pytest.raises(ValueError, match="expected"):
        call(pkg, dict(c, A=c["A"].cpu()))
    with pytest.raises(ValueError, match="lengths"):
        call(pkg, dict(c, lengths=torch.zeros(2, dtype=torch.int32, device=device)))
    big = torch.zeros(1, device=device).expand(1, 1, 1 << 22)
    with pytest.raises(Exception, match="2\\^22"):
        pkg.selective_scan(big, big, torch.zeros(1, 1, device=device).expand(1 << 22, 1), big[..., :1], big[..., :1])


def test_gradients_that_cannot_be_formed_are_refused_in_front(pkg, device):
    """B N G of 2^24: the call with gradients is refused before its forward runs, the one without them runs."""
    x = torch.full((1, 1, 16), 0.5, device=device).expand(1, 1 << 20, 16)
    A = -torch.ones(16, 1, device=device)
    rows = x[..., None]
    assert bool((pkg.selective_scan(x, x, A, rows, rows) > 0).all())
    with pytest.raises(pkg._lib.NativeLibraryError, match="gradients"):
        pkg.selective_scan(x, x, A.requires_grad_(True), rows, rows)


def step_call(pkg, c, rows, pool, **kw):
    return pkg.selective_scan_step(*(rows[k] for k in ("x", "delta")), c["A"], rows["B"], rows["C"], pool, skip=c.get("skip"),
                                   gate=rows.get("gate"), delta_bias=c.get("delta_bias"), softplus=c["softplus"], **kw)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,S,G", [(16, 16, None), (8, 8, 2), (100, 32, None), (7, 64, 7), (70, 5, 2), (1, 1, None), (33, 40, 3), (520, 16, None)])
@pytest.mark.parametrize("across", [False, True])
def test_steps(pkg, device, D, S, G, dtype, across):
    """Tokens one by one, in place and from pool to pool, with rows that pad the batch: the recurrence's values; slots that
    no row names stay as they are."""
    T = 5
    c = case(device, 3, T, D, S, dtype, G=G, seed=D)
    take, slots = [0, 2, 3], torch.tensor([4, -1, 0, 6, 7], device=device)
    pool = torch.full((7, D, S), 5.0, device=device)
    outs = []
    with torch.no_grad():
        pool[[4, 0, 6]] = c["initial"]
        for t in range(T):
            rows = {}
            for k in ("x", "delta", "gate", "B", "C"):
                rows[k] = torch.full((5, *c[k].shape[2:]), float("nan"), dtype=dtype, device=device)
                rows[k][take] = c[k][:, t]
            new = torch.full_like(pool, 5.0) if across else None
            out = step_call(pkg, c, rows, pool, slots=slots, new_state=new)
            assert not bool(out[[1, 4]].any())
            outs.append(out[take])
            pool = new if across else pool
    assert bool((pool[[1, 2, 3, 5]] == 5.0).all())
    ref = {k: f64(c[k]) for k in leaves_of(c)}
    want, wstate = selective_ref.selective_scan(**ref, softplus=True)
    off = scan_bounds(ref, True)
    within(torch.stack(outs, 1), want, off["y"], dtype, U)
    within(pool[[4, 0, 6]], wstate, off["state"], torch.float32, U)


@pytest.mark.parametrize("D,S", [(40, 16), (13, 5)])
def test_rows_of_one_slot_are_tokens_in_order(pkg, device, D, S):
    c = case(device, 1, 9, D, S, torch.bfloat16)
    rows = {k: c[k].detach()[0] for k in ("x", "delta", "gate", "B", "C")}
    slots = torch.tensor([2, 0, 2, -1, 2, 1, 0, 2, 4], dtype=torch.int32, device=device)
    start = torch.randn(4, D, S, device=device)
    one, many, across, new = (start.clone() for _ in range(4))
    with torch.no_grad():
        want = torch.cat([step_call(pkg, c, {k: v[i:i + 1] for k, v in rows.items()}, one, slots=slots[i:i + 1]) for i in range(9)])
        assert torch.equal(step_call(pkg, c, rows, many, slots=slots), want) and torch.equal(one, many)
        assert torch.equal(step_call(pkg, c, rows, across, slots=slots, new_state=new), want)
    assert torch.equal(new, one) and torch.equal(across, start)


def test_step_layouts_and_refusals(pkg, device):
    c = case(device, 1, 4, 16, 8, torch.bfloat16, parts=())
    rows = {k: c[k].detach()[0] for k in ("x", "delta", "B", "C")}
    start = torch.randn(6, 16, 8, device=device)
    a, b = start.clone(), start.clone()
    padded = torch.zeros(6, 17, 8, device=device)
    padded[:, :16] = start
    odd = torch.empty(start.numel() + 1, device=device)[1:].view(start.shape).copy_(start)
    with torch.no_grad():
        want = step_call(pkg, c, rows, a)
        strided = {k: torch.cat((v, v), -1)[..., :v.shape[-1]] for k, v in rows.items()}
        assert torch.equal(step_call(pkg, c, strided, b), want) and torch.equal(a, b)
        assert torch.equal(step_call(pkg, c, rows, padded[:, :16]), want) and torch.equal(padded[:, :16], a)
        assert torch.equal(step_call(pkg, c, rows, odd), want) and torch.equal(odd, a) and not bool(padded[:, 16:].any())
        with pytest.raises(ValueError, match="shares memory"):
            step_call(pkg, dict(c), dict(rows, x=b.view(torch.bfloat16)[0, :4]), b)
        with pytest.raises(ValueError, match="overlap"):
            step_call(pkg, c, rows, padded[:5, :16], new_state=padded[1:, :16])
        empty = {k: v[:0] for k, v in rows.items()}
        assert step_call(pkg, c, empty, b).shape == (0, 16)
        before = b.clone()
        out = step_call(pkg, c, rows, b, slots=torch.tensor([2 ** 32, -2 ** 33, 6, 3], device=device))
        assert not bool(out[:3].any()) and torch.equal(b[[0, 1, 2, 4, 5]], before[[0, 1, 2, 4, 5]]) and not torch.equal(b[3], before[3])
    with pytest.raises(RuntimeError, match="no gradients"):
        step_call(pkg, c, rows, b)


def test_step_slots_past_32_bits(pkg, device):
    """A pool of more than 2^32 elements: the last slots."""
    P, D, S = 9000, 8192, 64
    pool = torch.empty(P, D, S, device=device)
    small = torch.randn(2, D, S, device=device)
    pool[[P - 1, P - 2]] = small
    c = case(device, 1, 2, D, S, torch.bfloat16, parts=())
    rows = {k: c[k].detach()[0] for k in ("x", "delta", "B", "C")}
    with torch.no_grad():
        want = step_call(pkg, c, rows, small)
        assert torch.equal(step_call(pkg, c, rows, pool, slots=torch.tensor([P - 1, P - 2], device=device)), want)
    assert torch.equal(pool[[P - 1, P - 2]], small)
