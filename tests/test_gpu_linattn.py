"""GPU tests of decayed linear attention (linear_attention, linear_attention_step) against the float64 recurrence.

Error bound: fp32 sums of up to 64 products twice (scores, values), a decay weight (exp2 of an argument below 40 in
magnitude where the weight matters: 40 half steps, 2 for the instruction) and one product and sum for each chunk
and segment behind it: fewer than 400 half steps of fp32 in all, relative to the sum of the terms' absolute values.
Operands that a kernel splits into two bf16 parts keep 2^-16 (half a step of half a step, 2^-9 each, the two operands
of a product).  dlog_decay adds sum tau (o.do - k.dk) with tau below the segment length from its middle: the same
bound over those terms.
"""

import math

import pytest
import torch

from oracle import mixer_ref
from tests.mixer_cases import DTYPES, randn, within

pytestmark = pytest.mark.gpu
HD = 64


def slack(dtype):
    return 400 * 2.0 ** -24 + (0.0 if dtype == torch.float32 else 2.0 ** -15)


FP32 = 400 * 2.0 ** -24   # results that stay in fp32


def make(B, H, Hkv, N, dtype, seed, initial=False, lengths=None, decays=None, layout="token"):
    g = torch.Generator().manual_seed(seed)
    heads = (lambda n: randn(g, B, N, n, HD, dtype=dtype).transpose(1, 2)) if layout == "token" else (
        lambda n: randn(g, B, n, N, HD, dtype=dtype))
    x = dict(q=heads(H), k=heads(Hkv), v=heads(Hkv))
    at = torch.linspace(math.log(4.0), math.log(512.0), H)
    x["log_decay"] = torch.log1p(-torch.exp(-at)) if decays is None else torch.tensor(decays)
    x["initial"] = randn(g, B, H, HD, HD) if initial else None
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    x["dout"] = heads(H)
    x["dstate"] = randn(g, B, H, HD, HD)
    return x


def put(x, device):
    return {n: None if t is None else t.to(device) for n, t in x.items()}


def absolute(x):
    return {n: t if t is None or n in ("log_decay", "lengths") else t.abs() for n, t in x.items()}


def oracle(x, scale=0.125):
    args = (x["q"], x["k"], x["v"], x["log_decay"], scale)
    return mixer_ref.linear_attention(*args, x["initial"], x["lengths"])


def oracle_grads(x, scale=0.125, state=True):
    return mixer_ref.linear_attention_backward(x["q"], x["k"], x["v"], x["log_decay"], scale, x["dout"], x["initial"],
                                               x["lengths"], x["dstate"] if state else None)


def forward(pkg, d, **kw):
    return pkg.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], initial_state=d["initial"],
                                lengths=d["lengths"], **kw)


SHAPES = [
    # B, H, Hkv, N, initial, lengths
    (1, 1, 1, 1, False, None),
    (2, 3, 3, 1, True, None),
    (1, 2, 1, 7, True, None),
    (2, 2, 2, 63, False, None),
    (1, 4, 2, 64, True, None),
    (1, 2, 2, 65, True, None),
    (3, 4, 1, 130, True, [130, 0, 65]),
    (2, 2, 2, 200, False, [199, 64]),
    (4, 2, 2, 150, True, [-3, 1000, 128, 1]),
    (2, 64, 32, 300, False, [300, 257]),      # segments of 64
    (8, 32, 32, 300, True, None),              # segments of 256, the second with 44 tokens
    (9, 32, 8, 200, False, None),              # segments of 128, shared heads
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,N,initial,lengths", SHAPES)
def test_forward(pkg, device, B, H, Hkv, N, initial, lengths, dtype):
    if B * H * N > 40000 and dtype == torch.float16:
        pytest.skip("the two other types cover these segments")
    x = make(B, H, Hkv, N, dtype, seed=N + B, initial=initial, lengths=lengths)
    out, state = forward(pkg, put(x, device), return_state=True)
    assert out.dtype == dtype and out.transpose(1, 2).is_contiguous() and state.dtype == torch.float32
    want, wstate = oracle(x)
    terms, tstate = oracle(absolute(x))
    within(out, want, terms, dtype, slack(dtype))
    within(state, wstate, tstate, torch.float32, FP32)
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert not bool(out[b, :, min(max(n, 0), N):].any())
    alone = forward(pkg, put(x, device))
    assert torch.equal(alone, out)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,N,initial,lengths", SHAPES[:9] + [(2, 64, 32, 200, True, [200, 129])])
def test_gradients(pkg, device, B, H, Hkv, N, initial, lengths, dtype):
    x = make(B, H, Hkv, N, dtype, seed=3 * N + B, initial=initial, lengths=lengths)
    d = put(x, device)
    leaves = [n for n in ("q", "k", "v", "log_decay", "initial") if d[n] is not None]
    for n in leaves:
        d[n].requires_grad_(True)
    out, state = forward(pkg, d, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad((out, state), [d[n] for n in leaves], (d["dout"], d["dstate"]))))
    names = ("q", "k", "v", "log_decay", "initial")
    want, terms = dict(zip(names, oracle_grads(x))), dict(zip(names, oracle_grads(absolute(x))))
    for n in ("q", "k", "v"):
        assert got[n].dtype == dtype and got[n].transpose(1, 2).is_contiguous()
        within(got[n], want[n], terms[n], dtype, slack(dtype))
    if initial:
        within(got["initial"], want["initial"], terms["initial"], torch.float32, FP32)
    # tau (o.do) and tau (k.dk), tau up to 128 from the middle, and the states' products up to 256 of them: each of the
    # three no more than 256 times the sum of |q.dq| and |S||G|
    a = absolute(x)
    flow = (a["q"].double() * terms["q"]).sum((0, 2, 3)) + (oracle(a)[1] * a["dstate"].double()).sum((0, 2, 3))
    within(got["log_decay"], want["log_decay"], 3 * 256 * flow, torch.float32, slack(dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,N,lengths", [(13, 1, 1, None), (64, 8, 1, None), (3, 2, 200, [1, 0, 1]), (70, 8, 70, [1] * 70)])
def test_one_token_has_no_decay_gradient(pkg, device, B, H, N, lengths, dtype):
    """A sequence's first token onto an empty state: no decay stands in its output or its state, so the gradient is 0
    itself, in short segments and in long ones."""
    d = put(make(B, H, H, N, dtype, seed=B + N, lengths=lengths), device)
    d["log_decay"].requires_grad_(True)
    out, state = forward(pkg, d, return_state=True)
    g, = torch.autograd.grad((out, state), d["log_decay"], (d["dout"], d["dstate"]))
    assert torch.equal(g, torch.zeros_like(g))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,N,initial,lengths", [(1, 4, 2, 655, False, None), (2, 3, 3, 257, True, [257, 64]),
                                                       (1, 2, 1, 31, True, None), (16, 32, 32, 40, True, None)])
def test_decay_gradient_where_nothing_cancels(pkg, device, B, H, Hkv, N, initial, lengths, dtype):
    """Segments of one chunk add positive multiples of each share: the fp32 bound over the terms themselves."""
    x = make(B, H, Hkv, N, dtype, seed=N, initial=initial, lengths=lengths)
    d = put(x, device)
    d["log_decay"].requires_grad_(True)
    out, state = forward(pkg, d, return_state=True)
    g, = torch.autograd.grad((out, state), d["log_decay"], (d["dout"], d["dstate"]))
    within(g, oracle_grads(x)[3], oracle_grads(absolute(x))[3], torch.float32, FP32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("B,H,Hkv,N,lengths", [(2, 2, 1, 700, [700, 577]), (3, 1, 1, 512, [512, 65, 513]),
                                               (1, 1, 1, 9001, None), (2, 1, 1, 8300, [8193, 1100])])
def test_many_segments(pkg, device, B, H, Hkv, N, lengths, dtype):
    """More segments than one thread of the scan takes, and more than one pass of it: forward and gradients."""
    x = make(B, H, Hkv, N, dtype, seed=N, initial=True, lengths=lengths, decays=[-0.002] * H)
    d = put(x, device)
    names = ("q", "k", "v", "log_decay", "initial")
    for n in names:
        d[n].requires_grad_(True)
    out, state = forward(pkg, d, return_state=True)
    segments = -(-N // 64)
    # one more product and sum for each segment that a state has passed, on top of the module's bound
    more = segments * 2 * 2.0 ** -24
    want, wstate = oracle(x)
    terms, tstate = oracle(absolute(x))
    within(out, want, terms, dtype, slack(dtype) + more)
    within(state, wstate, tstate, torch.float32, FP32 + more)
    got = dict(zip(names, torch.autograd.grad((out, state), [d[n] for n in names], (d["dout"], d["dstate"]))))
    want, terms = dict(zip(names, oracle_grads(x))), dict(zip(names, oracle_grads(absolute(x))))
    for n in ("q", "k", "v"):
        within(got[n], want[n], terms[n], dtype, slack(dtype) + more)
    within(got["initial"], want["initial"], terms["initial"], torch.float32, FP32 + more)
    a = absolute(x)
    flow = (a["q"].double() * terms["q"]).sum((0, 2, 3)) + (oracle(a)[1] * a["dstate"].double()).sum((0, 2, 3))
    within(got["log_decay"], want["log_decay"], 3 * 512 * flow, torch.float32, slack(dtype) + more)


def test_gradients_with_parts_left_out(pkg, device):
    """Without dstate, without log_decay's or the initial state's gradient, and through the state alone."""
    x = make(2, 4, 2, 150, torch.float32, seed=5, initial=True)
    d = put(x, device)
    full = oracle_grads(x, state=False)
    terms = oracle_grads(absolute(x), state=False)
    d["q"].requires_grad_(True)
    d["initial"].requires_grad_(True)
    out = forward(pkg, d)
    dq, dS0 = torch.autograd.grad(out, (d["q"], d["initial"]), d["dout"])
    within(dq, full[0], terms[0], torch.float32, slack(torch.float32))
    within(dS0, full[4], terms[4], torch.float32, FP32)
    d = put(x, device)
    d["k"].requires_grad_(True)
    d["log_decay"].requires_grad_(True)
    _, state = forward(pkg, d, return_state=True)
    dk, dlg = torch.autograd.grad(state, (d["k"], d["log_decay"]), d["dstate"])
    none = dict(x, dout=torch.zeros_like(x["dout"]))
    want, terms = oracle_grads(none), oracle_grads(absolute(none))
    within(dk, want[1], terms[1], torch.float32, slack(torch.float32))
    a = absolute(x)
    flow = (oracle(a)[1] * a["dstate"].double()).sum((0, 2, 3))
    within(dlg, want[3], 3 * 256 * flow, torch.float32, FP32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("initial", [False, True])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("B,H,Hkv,N,lengths", [(2, 2, 1, 40, [40, 9]), (14, 32, 32, 100, [100, 64, 65, 0] + [77] * 10)])
def test_decay_gradient_of_a_single_segment(pkg, device, B, H, Hkv, N, lengths, state, initial, dtype):
    """One segment of one chunk and of two, with and without a state that enters (and needs no gradient) or leaves."""
    x = make(B, H, Hkv, N, dtype, seed=N + state, initial=initial, lengths=lengths)
    d = put(x, device)
    names = ("q", "k", "v", "log_decay")
    for n in names:
        d[n].requires_grad_(True)
    out, left = forward(pkg, d, return_state=True)
    outs, ups = ((out, left), (d["dout"], d["dstate"])) if state else ((out,), (d["dout"],))
    got = torch.autograd.grad(outs, [d[n] for n in names], ups)
    a = absolute(x)
    want, terms = oracle_grads(x, state=state), oracle_grads(a, state=state)
    for i in range(3):
        within(got[i], want[i], terms[i], dtype, slack(dtype))
    # as in test_gradients
    flow = (a["q"].double() * terms[0]).sum((0, 2, 3)) + (oracle(a)[1] * a["dstate"].double()).sum((0, 2, 3))
    within(got[3], want[3], 3 * 256 * flow, torch.float32, slack(dtype))


def test_gradients_match_differences(pkg, device):
    """The output is linear in q, in k and in v and the state enters linearly: a central difference of any step is
    exact up to rounding.  log_decay takes a step that stays below 0; what its difference leaves out is the float64
    oracle's difference less the oracle's gradient."""
    x = make(1, 4, 2, 140, torch.float32, seed=9, initial=True)
    d = put(x, device)
    names = ("q", "k", "v", "log_decay", "initial")
    for n in names:
        d[n].requires_grad_(True)

    def loss(t):
        out, state = forward(pkg, t, return_state=True)
        return (out.double() * d["dout"].double()).sum() + (state.double() * d["dstate"].double()).sum()

    def exact_loss(t):
        out, state = oracle(t)
        return float((out * x["dout"].double()).sum() + (state * x["dstate"].double()).sum())

    grads = torch.autograd.grad(loss(d), [d[n] for n in names])
    exact = dict(zip(names, oracle_grads(x)))
    a = absolute(x)
    out, state = oracle(a)
    size = float((out * a["dout"].double()).sum() + (state * a["dstate"].double()).sum())
    g = torch.Generator().manual_seed(1)
    for n, grad in zip(names, grads):
        way = torch.rand(4, generator=g) if n == "log_decay" else randn(g, *d[n].shape)
        h = 2.0 ** -10 if n == "log_decay" else 0.5
        moved = [x[n] + s * h * way for s in (1, -1)]   # the fp32 values that both sides see
        with torch.no_grad():
            up, down = (loss(dict(d, **{n: t.to(device)})) for t in moved)
        numeric = float(up - down) / (2 * h)
        analytic = float((grad.double().cpu() * way.double()).sum())
        left_out = (exact_loss(dict(x, **{n: moved[0]})) - exact_loss(dict(x, **{n: moved[1]}))) / (2 * h) - float(
            (exact[n].double() * way.double()).sum())
        # two losses of 400 half steps of their terms; those terms grow with the step, by less than 4 for |way| < 6
        bound = abs(left_out) + 2 * FP32 * 4 * size / (2 * h)
        assert abs(numeric - analytic) <= bound, n


def test_decay_edges(pkg, device):
    """-inf (the token alone), the lowest fp32, 0 and values above 0 (a plain running sum), 1e-8 from 0."""
    low = torch.finfo(torch.float32).min
    x = make(1, 5, 5, 150, torch.float32, seed=2, initial=True, decays=[-math.inf, low, 0.0, 0.7, -1e-8])
    d = put(x, device)
    d["log_decay"].requires_grad_(True)
    out, state = forward(pkg, d, return_state=True)
    want, wstate = oracle(x)
    terms, tstate = oracle(absolute(x))
    within(out, want, terms, torch.float32, slack(torch.float32))
    within(state, wstate, tstate, torch.float32, FP32)
    (dlg,) = torch.autograd.grad((out, state), d["log_decay"], (d["dout"], d["dstate"]))
    assert bool(torch.isfinite(dlg).all()) and float(dlg[3]) == 0.0


def test_padding_is_not_read(pkg, device):
    """NaN and infinities behind the lengths change nothing: not the results, not the gradients."""
    lengths = [100, 33, 0]
    x = make(3, 4, 2, 130, torch.bfloat16, seed=4, initial=True, lengths=lengths)
    results = []
    for bad in (0.0, math.nan, math.inf):
        d = put(x, device)
        for n in ("q", "k", "v", "dout"):
            for b, m in enumerate(lengths):
                d[n][b, :, m:] = bad
        leaves = [d[n].requires_grad_(True) for n in ("q", "k", "v", "log_decay", "initial")]
        out, state = forward(pkg, d, return_state=True)
        results.append([out, state, *torch.autograd.grad((out, state), leaves, (d["dout"], d["dstate"]))])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    for n, grad in zip("qkv", results[0][2:5]):
        for b, m in enumerate(lengths):
            assert not bool(grad[b, :, m:].any()), n


def test_layouts_agree_bit_for_bit(pkg, device):
    """Head-major tensors, views of one fused projection, rows off 16-byte alignment and int64 lengths."""
    x = make(2, 4, 2, 90, torch.bfloat16, seed=6, lengths=[90, 71])
    d = put(x, device)
    want = forward(pkg, d)
    major = dict(d, **{n: d[n].contiguous() for n in ("q", "k", "v")}, lengths=d["lengths"].long())
    assert torch.equal(forward(pkg, major), want)
    fused = torch.cat([d[n].transpose(1, 2).reshape(2, 90, -1) for n in ("q", "k", "v")], -1)
    parts = [t.unflatten(-1, (-1, HD)).transpose(1, 2) for t in fused.split([256, 128, 128], -1)]
    assert torch.equal(forward(pkg, dict(d, **dict(zip("qkv", parts)))), want)
    one = d["k"][:, :, :1].expand(-1, -1, 90, -1)          # one key for every token: rows a stride of 0 apart
    assert torch.equal(forward(pkg, dict(d, k=one)), forward(pkg, dict(d, k=one.contiguous())))
    over = torch.randn(90 * 8 + 64, device=device).bfloat16().as_strided((2, 4, 90, 64), (0, 0, 8, 1))   # overlapping rows
    assert torch.equal(forward(pkg, dict(d, q=over)), forward(pkg, dict(d, q=over.contiguous())))
    single = torch.randn(2, 4, 1, 64, device=device).bfloat16()
    tight = single.as_strided((2, 4, 1, 64), (256, 64, 0, 1))
    alone = dict(d, k=d["k"][:, :, :1], v=d["v"][:, :, :1], lengths=None)
    assert torch.equal(forward(pkg, dict(alone, q=tight)), forward(pkg, dict(alone, q=single)))
    odd = torch.empty(2, 4, 90, 67, device=device, dtype=torch.bfloat16)[..., 1:65]
    odd.copy_(d["q"])
    assert torch.equal(forward(pkg, dict(d, q=odd)), want)


def test_sequences_join_through_their_state(pkg, device):
    """A prompt in two calls, the second from the first one's state, and then token by token."""
    x = make(2, 4, 2, 200, torch.float32, seed=8)
    d = put(x, device)
    want, wstate = oracle(x)
    terms, tstate = oracle(absolute(x))
    first = dict(d, **{n: d[n][:, :, :77] for n in ("q", "k", "v")})
    a, state = forward(pkg, first, return_state=True)
    second = dict(d, **{n: d[n][:, :, 77:150] for n in ("q", "k", "v")}, initial=state)
    b, state = forward(pkg, second, return_state=True)
    steps = [pkg.linear_attention_step(d["q"][:, :, t], d["k"][:, :, t], d["v"][:, :, t], d["log_decay"], state)
             for t in range(150, 200)]
    got = torch.cat([a, b, torch.stack(steps, 2)], 2)
    # the states pass through 50 single steps: three roundings each on top
    within(got, want, terms, torch.float32, slack(torch.float32) + 150 * 2.0 ** -24)
    within(state, wstate, tstate, torch.float32, FP32 + 150 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("S,H,Hkv,pool", [(1, 1, 1, 1), (3, 4, 2, 7), (37, 8, 1, 64)])
def test_step(pkg, device, S, H, Hkv, pool, dtype):
    """Against the recurrence, in place and from one pool into another; padded and out-of-range rows touch nothing."""
    g = torch.Generator().manual_seed(S)
    q, k, v = (randn(g, S, n, HD, dtype=dtype) for n in (H, Hkv, Hkv))
    lg = -torch.rand(H, generator=g)
    state = randn(g, pool, H, HD, HD)
    slots = torch.randperm(pool, generator=g)[:S].to(torch.int32)
    if S > 2:
        slots[1], slots[S - 1] = -1, pool + 5
    dev = [t.to(device) for t in (q, k, v, lg, state, slots)]
    other = torch.full_like(dev[4], 7.0)
    out = pkg.linear_attention_step(*dev[:4], dev[4], slots=dev[5], new_state=other)
    assert torch.equal(dev[4].cpu(), state)
    again = torch.empty_like(out)
    assert pkg.linear_attention_step(*dev[:4], dev[4], slots=dev[5].long(), out=again) is again
    assert torch.equal(again, out)
    for s in range(S):
        slot = int(slots[s])
        if not 0 <= slot < pool:
            assert not bool(out[s].any())
            continue
        args = [t[s][None, :, None] for t in (q, k, v)]
        want, wstate = mixer_ref.linear_attention(*args, lg, 0.125, state[slot][None])
        terms, tstate = mixer_ref.linear_attention(*(t.abs() for t in args), lg, 0.125, state[slot][None].abs())
        # a decay weight (42 half steps), one product and sum for the state, 64 of them for the output
        within(out[s], want[0, :, 0], terms[0, :, 0], dtype, 150 * 2.0 ** -24)
        within(other[slot], wstate[0], tstate[0], torch.float32, 50 * 2.0 ** -24)
    touched = [int(s) for s in slots if 0 <= int(s) < pool]
    rest = [i for i in range(pool) if i not in touched]
    assert torch.equal(dev[4][rest].cpu(), state[rest]) and bool((other[rest] == 7.0).all())
    assert torch.equal(dev[4][touched], other[touched])


def test_step_rows_of_one_slot_follow_each_other(pkg, device):
    """The same slot several times in a call: consecutive tokens, bit for bit the calls one by one."""
    g = torch.Generator().manual_seed(3)
    S, H, Hkv, pool = 300, 4, 2, 5
    q, k, v = (randn(g, S, n, HD, dtype=torch.bfloat16).to(device) for n in (H, Hkv, Hkv))
    lg = -torch.rand(H, generator=g).to(device)
    state = randn(g, pool, H, HD, HD).to(device)
    slots = torch.tensor([(i * i) % 6 - 1 for i in range(S)], dtype=torch.int32, device=device)   # -1 among them
    together, single = state.clone(), state.clone()
    out = pkg.linear_attention_step(q, k, v, lg, together, slots=slots)
    for s in range(S):
        one = pkg.linear_attention_step(q[s:s + 1], k[s:s + 1], v[s:s + 1], lg, single, slots=slots[s:s + 1])
        assert torch.equal(one[0], out[s])
    assert torch.equal(together, single)


def test_step_strided_pool_and_default_slots(pkg, device):
    """A pool of every layer, one layer's slots a stride apart; without slots row s works on state s."""
    g = torch.Generator().manual_seed(4)
    q, k, v = (randn(g, 3, 2, HD).to(device) for _ in range(3))
    lg = -torch.rand(2, generator=g).to(device)
    layers = randn(g, 4, 3, 2, HD, HD).to(device)   # [slots, layers, H, 64, 64]
    want = layers[:, 1].contiguous()
    a = pkg.linear_attention_step(q, k, v, lg, want)
    before = layers.clone()
    b = pkg.linear_attention_step(q, k, v, lg, layers[:, 1])
    assert torch.equal(a, b) and torch.equal(layers[:, 1], want) and torch.equal(layers[:, 0], before[:, 0])
    assert torch.equal(layers[:, 2], before[:, 2])
    with pytest.raises(ValueError, match="overlap"):
        pkg.linear_attention_step(q, k, v, lg, layers[:3, 1], new_state=layers[1:, 1])
    with pytest.raises(RuntimeError, match="no gradients"):
        pkg.linear_attention_step(q.clone().requires_grad_(True), k, v, lg, want)


def test_empty_calls(pkg, device):
    """No tokens, no sequences, no rows: the state that enters leaves, gradients are zero."""
    x = make(2, 4, 2, 0, torch.bfloat16, seed=1, initial=True)
    d = put(x, device)
    leaves = [d[n].requires_grad_(True) for n in ("q", "k", "v", "log_decay", "initial")]
    out, state = forward(pkg, d, return_state=True)
    assert out.shape == (2, 4, 0, HD) and torch.equal(state.detach(), d["initial"].detach())
    grads = torch.autograd.grad((out, state), leaves, (d["dout"], d["dstate"]))
    assert torch.equal(grads[4], d["dstate"]) and not bool(grads[3].any())
    x = make(0, 4, 2, 5, torch.bfloat16, seed=1)
    d = put(x, device)
    leaves = [d[n].requires_grad_(True) for n in ("q", "log_decay")]
    out, state = forward(pkg, d, return_state=True)
    assert out.shape == (0, 4, 5, HD) and state.shape == (0, 4, HD, HD)
    assert not bool(torch.autograd.grad(out, leaves, d["dout"])[1].any())
    q, k, v = (torch.empty(0, n, HD, device=device) for n in (4, 2, 2))
    assert pkg.linear_attention_step(q, k, v, torch.zeros(4, device=device), torch.zeros(2, 4, HD, HD, device=device)).shape == (0, 4, HD)


def test_same_bits_every_time_and_second_derivatives_are_refused(pkg, device):
    x = make(3, 8, 2, 300, torch.bfloat16, seed=7, initial=True)

    def once():
        d = put(x, device)
        leaves = [d[n].requires_grad_(True) for n in ("q", "k", "v", "log_decay", "initial")]
        out, state = forward(pkg, d, return_state=True)
        return [out, state, *torch.autograd.grad((out, state), leaves, (d["dout"], d["dstate"]))]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)
    d = put(x, device)
    d["q"].requires_grad_(True)
    (dq,) = torch.autograd.grad(forward(pkg, d), d["q"], d["dout"].requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), d["dout"])


def test_long_sequence_against_its_parts(pkg, device):
    """70,001 tokens in one call and in two: the states' offsets pass a segment count of one call's own."""
    g = torch.Generator().manual_seed(11)
    N, cut = 70001, 40007
    q, k, v = (randn(g, 1, N, 2, HD, dtype=torch.bfloat16).to(device).transpose(1, 2) for _ in range(3))
    lg = torch.tensor([-0.01, -0.0005], device=device)
    out, state = pkg.linear_attention(q, k, v, lg, return_state=True)
    a, mid = pkg.linear_attention(q[:, :, :cut], k[:, :, :cut], v[:, :, :cut], lg, return_state=True)
    b, end = pkg.linear_attention(q[:, :, cut:], k[:, :, cut:], v[:, :, cut:], lg, initial_state=mid, return_state=True)
    # both sides round once to bf16 and differ by the order of fp32 sums: terms about sqrt(2000) wide
    both = torch.cat([a, b], 2).float()
    assert float((out.float() - both).abs().max()) <= 2 * 2.0 ** -8 * float(both.abs().max())
    assert float((state - end).abs().max()) <= 1e-5 * float(end.abs().max())


def test_graph_replays_and_other_streams(pkg, device):
    """Forward, backward and step captured once and replayed with eager work between; the same on a second stream."""
    x = make(2, 4, 2, 200, torch.bfloat16, seed=12, initial=True)
    d = put(x, device)
    pool = d["initial"].clone()

    def work():
        la = pkg.linattn
        out, state, states = la.attention_forward(d["q"], d["k"], d["v"], d["log_decay"], d["initial"], None, 0.125, True)
        grads = la.attention_backward(d["dout"], d["dstate"], d["q"], d["k"], d["v"], d["log_decay"], d["initial"], None,
                                      0.125, states, state, True, True)
        step = pkg.linear_attention_step(d["q"][:, :, 0], d["k"][:, :, 0], d["v"][:, :, 0], d["log_decay"], d["initial"],
                                         new_state=pool)
        return [out, state, *grads, step, pool]

    want = [t.clone() for t in work()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [t.clone() for t in work()]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    q = d["q"].clone()
    for rep in range(3):
        d["q"].copy_(q * (rep + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, work())), rep
        torch.cuda.synchronize()


def test_compiled_matches_eager(pkg, device):
    x = make(2, 4, 2, 130, torch.bfloat16, seed=13, initial=True)

    def step(q, k, v, lg, S0):
        out, state = pkg.linear_attention(q, k, v, lg, initial_state=S0, return_state=True)
        return (out.float() ** 2).sum() + state.sum()

    results = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        d = put(x, device)
        leaves = [d[n].requires_grad_(True) for n in ("q", "k", "v", "log_decay", "initial")]
        loss = fn(*leaves)
        loss.backward()
        results.append([loss.detach(), *(t.grad for t in leaves)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
