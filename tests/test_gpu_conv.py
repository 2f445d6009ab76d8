"""GPU tests of causal_conv and causal_conv_step against the float64 sums over the taps.

Bounds, in u = 2^-24: p is a chain of W fused steps on the bias (W + 1 with the bias's own); silu and its slope as in
selective_cases.  dx is a chain of W products dp w and the final state's gradient; a weight's gradient is a chain of a
strip's up to 64 tokens and a workgroup's 8 strips in fp32, then 64-bit sums.
"""

import pytest
import torch

from oracle import selective_ref
from tests.mixer_cases import DTYPES, randn
from tests.selective_cases import U, conv_strips, f64, silu_off, slope_off, within

pytestmark = pytest.mark.gpu


def case(device, B, N, D, W, dtype, seed=0, bias=True, initial=True, lengths=None, wtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=randn(g, B, N, D, dtype=dtype), weight=randn(g, D, W, dtype=wtype), bias=randn(g, D, dtype=wtype) if bias else None,
             initial=randn(g, B, W - 1, D, dtype=dtype) if initial else None)
    c = {k: None if v is None else v.to(device).requires_grad_(True) for k, v in c.items()}
    c["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    c["dy"], c["dstate"] = randn(g, B, N, D, dtype=dtype).to(device), randn(g, B, W - 1, D, dtype=dtype).to(device)
    return c


def call(pkg, c, activation):
    return pkg.causal_conv(c["x"], c["weight"], c["bias"], activation=activation, initial_state=c["initial"], lengths=c["lengths"],
                           return_state=True)


def check(pkg, c, activation, use_state=True):
    y, state = call(pkg, c, activation)
    dtype, W = c["x"].dtype, c["weight"].shape[1]
    names = [k for k in ("x", "weight", "bias", "initial") if c[k] is not None]
    outs, ups = ([y, state], [c["dy"], c["dstate"]]) if use_state else ([y], [c["dy"]])
    grads = dict(zip(names, torch.autograd.grad(outs, [c[k] for k in names], ups)))
    leaves = {k: f64(c[k]).requires_grad_(True) for k in names}
    lengths = None if c["lengths"] is None else c["lengths"].cpu()
    args = [leaves["x"], leaves["weight"], leaves.get("bias"), activation, leaves.get("initial"), lengths]
    wy, wstate = selective_ref.causal_conv(*args)
    pre = wy if activation is None else selective_ref.causal_conv(*args[:3], None, *args[4:])[0]
    size = selective_ref.causal_conv(*(None if t is None else t.detach().abs() for t in args[:3]), None,
                                     None if args[4] is None else args[4].detach().abs(), lengths)[0]
    wants = dict(zip(names, torch.autograd.grad([wy, wstate][:len(outs)], [leaves[k] for k in names],
                                                [f64(u) for u in ups], allow_unused=True)))
    p, p_off = pre.detach(), (W + 1) * size
    y_off = p_off if activation is None else silu_off(p, p_off)
    assert torch.equal(f64(state), wstate.detach())
    within(y, wy.detach(), y_off, dtype, U)
    B, N, D = p.shape
    count = torch.full((B,), N) if lengths is None else lengths.clamp(0, N)
    alive = (torch.arange(N)[None] < count[:, None]).double()[..., None]
    assert not bool((f64(y) * (1 - alive)).any())
    e = torch.sigmoid(p)
    slope = torch.ones_like(p) if activation is None else (e * (1 + p * (1 - e))).abs()
    dp = f64(c["dy"]).abs() * slope * alive
    dp_off = f64(c["dy"]).abs() * (0 if activation is None else slope_off(p, p_off) + 2 * slope) * alive
    w = f64(c["weight"]).abs()
    front = torch.zeros(B, W - 1, D, dtype=torch.float64) if c["initial"] is None else f64(c["initial"]).abs()
    dwide, wide = torch.zeros(B, N + W - 1, D, dtype=torch.float64), torch.cat((front, f64(c["x"]).abs()), 1)
    dw_off = torch.zeros(D, W, dtype=torch.float64)
    for j in range(W):
        dwide[:, j:j + N] += (dp_off + (W + 2) * dp) * w[:, j]
        dw_off[:, j] = (wide[:, j:j + N] * (dp_off + 76 * dp)).sum((0, 1))
    if use_state:
        for b in range(B):
            dwide[b, int(count[b]):int(count[b]) + W - 1] += 2 * f64(c["dstate"][b]).abs()
    offs = dict(x=dwide[:, W - 1:], initial=dwide[:, :W - 1], weight=dw_off, bias=(dp_off + 76 * dp).sum((0, 1)))
    for k in names:
        want = wants[k] if wants[k] is not None else torch.zeros_like(leaves[k])
        within(grads[k], want.detach(), offs[k], c[k].dtype, U)
    return grads


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("W", range(1, 9))
@pytest.mark.parametrize("activation", [None, "silu"])
def test_widths(pkg, device, W, dtype, activation):
    check(pkg, case(device, 2, 37, 24, W, dtype, W), activation)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [0, 1, 2, 3, 15, 16, 17, 65, 200])
@pytest.mark.parametrize("D", [1, 3, 4, 7, 8, 9, 100, 260])
def test_sizes(pkg, device, N, D, dtype):
    """Token counts around the strips', channel counts below, at and beside whole vectors."""
    check(pkg, case(device, 2, N, D, 4, dtype, N * 1000 + D), "silu")


@pytest.mark.parametrize("B,N,D", [(40, 700, 40), (3, 4000, 520), (300, 5, 8)])
def test_longer_strips_and_many_sequences(pkg, device, B, N, D):
    check(pkg, case(device, B, N, D, 3, torch.bfloat16, initial=False), "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,N,D,W,activation,strip,lengths", [
    (4, 57400, 12, 4, "silu", 64, [57400, 19200, 19201, 33]), (4, 57400, 8, 3, None, 64, [57399, 64, 63, 57345]),
    (2, 57400, 12, 8, "silu", 32, [31999, 32001]), (2300, 100, 9, 4, "silu", 64, None)])
def test_strips_of_32_and_64_tokens(pkg, device, B, N, D, W, activation, strip, lengths, dtype):
    """The strips of large batches, forward and backward: sequences that end at a strip's end, beside it and inside, strips
    longer than what is left of a sequence."""
    assert conv_strips(B, N, D, dtype) == (strip, strip)
    check(pkg, case(device, B, N, D, W, dtype, seed=D, lengths=lengths), activation)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("W", [1, 2, 4, 8])
def test_lengths(pkg, device, W, initial, dtype):
    """Sequences that end anywhere, none of whose tokens count, and fewer than the taps."""
    lengths = [40, 0, 1, 2, 17, -3, 99, 3]
    check(pkg, case(device, 8, 40, 20, W, dtype, W, initial=initial, lengths=lengths), "silu")


def test_parts_and_table_types(pkg, device):
    for wtype in DTYPES:
        check(pkg, case(device, 2, 30, 16, 4, torch.bfloat16, wtype=wtype), "silu")
    check(pkg, case(device, 2, 30, 16, 4, torch.float16, bias=False, initial=False), None, use_state=False)


def test_values_behind_the_lengths_are_not_used(pkg, device):
    """NaN and infinities behind the end, in rows and their gradients: the bits of zeros there."""
    for lengths in ([20, 0, 7], [0, 0, 0]):
        c = case(device, 3, 33, 24, 4, torch.bfloat16, lengths=lengths)
        results = []
        for fill in (0.0, float("nan"), float("inf")):
            dead = torch.arange(33, device=device)[None] >= c["lengths"][:, None]
            d = dict(c, x=c["x"].detach().masked_fill(dead[..., None], fill).requires_grad_(True),
                     dy=c["dy"].masked_fill(dead[..., None], fill))
            y, s = call(pkg, d, "silu")
            results.append([y, s, *torch.autograd.grad([y, s], [d[k] for k in ("x", "weight", "bias", "initial")], [d["dy"], c["dstate"]])])
        for other in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(other, results[0]))


def test_layouts_give_the_same_bits(pkg, device):
    g = torch.Generator().manual_seed(1)
    wide = randn(g, 3, 50, 80, dtype=torch.bfloat16).to(device)
    w, c, front = (randn(g, *s).to(device) for s in ((32, 4), (32,), (3, 3, 32)))
    front = front.bfloat16()
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t)   # noqa: E731
    for x in (wide[..., 16:48], wide[..., 5:37], wide.transpose(0, 1)[:3, :, :32], wide[:1, :, :32].expand(3, 50, 32),
              wide[:, ::2, 32:64], wide[:, :1, :32].expand(3, 20, 32), wide[..., ::2][..., :32]):
        a = pkg.causal_conv(x, w, c, activation="silu", return_state=True)
        b = pkg.causal_conv(x.contiguous(), w, c, activation="silu", return_state=True)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    x = wide[..., :32].contiguous()
    a = pkg.causal_conv(x, w, c, initial_state=front, return_state=True)
    b = pkg.causal_conv(odd(x), odd(w.T.contiguous()).T, odd(c), initial_state=odd(front), return_state=True)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_parts_of_a_sequence(pkg, device):
    """A sequence in two calls, the state between them: the bits of one call."""
    c = case(device, 2, 60, 40, 5, torch.float16)
    with torch.no_grad():
        y, s = call(pkg, c, "silu")
        parts, state = [], c["initial"]
        for a, b in ((0, 2), (2, 3), (3, 60)):
            z, state = pkg.causal_conv(c["x"][:, a:b], c["weight"], c["bias"], activation="silu", initial_state=state, return_state=True)
            parts.append(z)
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(state, s)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D,W", [(1, 1), (5, 4), (8, 2), (100, 4), (260, 8), (2100, 4)])
@pytest.mark.parametrize("across", [False, True])
def test_steps_are_the_sequence(pkg, device, D, W, dtype, across):
    """Tokens one by one against a pool, in place and from pool to pool: the bits of the whole sequence's call.  Slots the
    rows do not name stay as they are."""
    c = case(device, 3, 6, D, W, dtype, initial=True)
    with torch.no_grad():
        want, final = call(pkg, c, "silu")
        pool = torch.full((7, W - 1, D), 5.0, dtype=dtype, device=device)
        slots = torch.tensor([4, -1, 0, 6, 7], device=device)
        pool[[4, 0, 6]] = c["initial"]
        old = pool.clone()
        for t in range(6):
            x = torch.zeros(5, D, dtype=dtype, device=device)
            x[[0, 2, 3]] = c["x"][:, t]
            new = torch.full_like(pool, 5.0) if across else None
            out = pkg.causal_conv_step(x, c["weight"], c["bias"], pool, activation="silu", slots=slots, new_state=new)
            assert torch.equal(out[[0, 2, 3]], want[:, t]) and not bool(out[[1, 4]].any())
            pool = new if across else pool
    assert torch.equal(pool[[4, 0, 6]], final) and torch.equal(pool[[1, 2, 3, 5]], old[[1, 2, 3, 5]])


def test_rows_of_one_slot_are_tokens_in_order(pkg, device):
    """Several rows of a slot, between others: the steps one after another."""
    g = torch.Generator().manual_seed(2)
    x, w, pool = randn(g, 9, 40).to(device), randn(g, 40, 4).to(device), randn(g, 4, 3, 40).to(device)
    slots = torch.tensor([2, 0, 2, -1, 2, 1, 0, 2, 4], dtype=torch.int32, device=device)
    one, many = pool.clone(), pool.clone()
    want = torch.cat([pkg.causal_conv_step(x[i:i + 1], w, None, one, slots=slots[i:i + 1]) for i in range(9)])
    assert torch.equal(pkg.causal_conv_step(x, w, None, many, slots=slots), want) and torch.equal(one, many)
    new = pool.clone()
    assert torch.equal(pkg.causal_conv_step(x, w, None, pool, slots=slots, new_state=new), want) and torch.equal(new, one)


def test_step_refusals_and_wide_pools(pkg, device):
    pool = torch.zeros(8, 6, 40, device=device)
    x, w = torch.randn(3, 40, device=device), torch.randn(40, 4, device=device)
    padded = pool[:, :3]   # slots further apart than they are long
    out = pkg.causal_conv_step(x, w, None, padded)
    assert torch.equal(out, pkg.causal_conv_step(x, w, None, torch.zeros(8, 3, 40, device=device))) and not bool(pool[:, 3:].any())
    with pytest.raises(ValueError, match="shares memory"):
        pkg.causal_conv_step(pool[:3, 1], w, None, pool[:, :3])
    with pytest.raises(ValueError, match="overlap"):
        pkg.causal_conv_step(x, w, None, pool[:7, :3], new_state=pool[1:, :3])
    with pytest.raises(ValueError, match="expected"):
        pkg.causal_conv_step(x, w.cpu(), None, padded)
    with pytest.raises(RuntimeError, match="no gradients"):
        pkg.causal_conv_step(x, w.requires_grad_(True), None, padded)
    assert pkg.causal_conv_step(x[:0], w.detach(), None, padded).shape == (0, 40)
    wide = torch.tensor([2 ** 32 + 1, -2 ** 32, 2], device=device)
    before = pool.clone()
    out = pkg.causal_conv_step(x, w.detach(), None, padded, slots=wide)
    assert not bool(out[:2].any()) and torch.equal(pool[[0, 1]], before[[0, 1]])


def test_second_derivative_and_tangents_are_refused(pkg, device):
    import torch.autograd.forward_ad as fw
    x, w = torch.randn(1, 5, 8, device=device, requires_grad=True), torch.randn(8, 3, device=device)
    g, = torch.autograd.grad(pkg.causal_conv(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="first order"):
        g.sum().backward()
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        pkg.causal_conv(fw.make_dual(x.detach(), x.detach()), w)


def test_far_rows(pkg, device):
    """Tokens and sequences whose offsets pass 2^31 elements."""
    buf = torch.empty((1 << 31) + (1 << 23), dtype=torch.bfloat16, device=device)
    x = buf.as_strided((2, 4, 40), ((1 << 31) - (1 << 20), 1 << 20, 1)).normal_()
    w = torch.randn(40, 3, device=device)
    assert torch.equal(pkg.causal_conv(x, w), pkg.causal_conv(x.clone(), w))


def test_same_bits_graph_and_compile(pkg, device):
    c = case(device, 3, 90, 72, 4, torch.bfloat16, lengths=[90, 11, 0])
    names = ("x", "weight", "bias", "initial")

    def work(x, weight, bias, initial):
        y, s = pkg.causal_conv(x, weight, bias, activation="silu", initial_state=initial, lengths=c["lengths"], return_state=True)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], [x, weight, bias, initial], [c["dy"], c["dstate"]])]

    rows, slots = c["x"].detach()[:, 0].contiguous(), torch.tensor([1, 1, -1], device=device)
    start = torch.randn(2, 3, 72, device=device).bfloat16()

    def step(pool, rows):
        with torch.no_grad():
            return pkg.causal_conv_step(rows, c["weight"], c["bias"], pool, activation="silu", slots=slots)

    eager = lambda: [t.clone() for t in work(*(c[k] for k in names))]   # noqa: E731
    want = eager()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(eager(), want))
    f = torch.compile(lambda x, w, b, i: pkg.causal_conv(x, w, b, activation="silu", initial_state=i, lengths=c["lengths"],
                                                         return_state=True), backend="aot_eager", fullgraph=True)
    out = f(*(c[k] for k in names))
    got = [*out, *torch.autograd.grad(out, [c[k] for k in names], [c["dy"], c["dstate"]])]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pools = [start.clone(), start.clone()]
    a, b = step(pools[0], rows), torch.compile(step, backend="aot_eager", fullgraph=True)(pools[1], rows)
    assert torch.equal(a, b) and torch.equal(*pools) and not torch.equal(pools[0], start)
    del out, got
    torch.cuda.synchronize()
    graph, pool = torch.cuda.CUDAGraph(), start.clone()
    with torch.cuda.graph(graph):
        outs = work(*(c[k] for k in names))
        out = step(pool, rows)
    other = start.clone()
    for rep in range(3):
        with torch.no_grad():
            c["x"].mul_(1 + rep)
            rows.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, eager())), rep
        assert torch.equal(out, step(other, rows)) and torch.equal(pool, other), rep
