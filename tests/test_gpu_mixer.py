"""GPU tests of the mixer's operators together, as a layer runs them: layer norm, q, k and v of one row, a norm of each
head, rotary positions, decayed linear attention, a norm of each head's output; trained in one call and served as a
prompt and single tokens.

Each stage is compared with its float64 oracle on the values that reached it, forward and backward, so that the bounds
are those of the operators alone (derived in their own test files).
"""

import math

import pytest
import torch

from oracle import mixer_ref
from tests.mixer_cases import DTYPES, randn, within
from tests.test_gpu_linattn import FP32, HD
from tests.test_gpu_linattn import slack as attention_slack
from tests.test_gpu_norm import steps
from tests.test_gpu_rotary import slack as rotary_slack
from tests.test_gpu_rotary import terms as rotary_terms

pytestmark = pytest.mark.gpu
H, HKV = 4, 2
WIDTH = (H + 2 * HKV) * HD


def make(B, N, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    scale = lambda *shape: 1 + 0.2 * randn(g, *shape)   # noqa: E731
    return dict(x=randn(g, B, N, WIDTH, dtype=dtype), w=scale(WIDTH), b=0.1 * randn(g, WIDTH), wq=scale(H, HD),
                wk=scale(HKV, HD), wo=scale(H, HD), bo=0.1 * randn(g, H, HD),
                log_decay=torch.log1p(-torch.exp(-torch.linspace(math.log(4.0), math.log(256.0), H)))), randn(
                    g, B, N, H, HD, dtype=dtype)


PARAMETERS = ("x", "w", "b", "wq", "wk", "wo", "bo", "log_decay")


def split(y):
    """q [.., H, 64], k and v [.., HKV, 64] of a row."""
    q, k, v = y.split([H * HD, HKV * HD, HKV * HD], -1)
    heads = lambda t: t.unflatten(-1, (t.shape[-1] // HD, HD))   # noqa: E731
    return heads(q), heads(k), heads(v)


def layer(pkg, p, positions, plan, lengths):
    s = {"y": pkg.layer_norm(p["x"], p["w"], p["b"])}
    s["q"], s["k"], s["v"] = split(s["y"])
    s["qn"], s["kn"] = pkg.layer_norm(s["q"], p["wq"]), pkg.layer_norm(s["k"], p["wk"])
    s["qr"], s["kr"] = pkg.rotary_embed(s["qn"].transpose(1, 2), s["kn"].transpose(1, 2), positions, plan)
    s["vt"] = s["v"].transpose(1, 2)
    s["out"], s["state"] = pkg.linear_attention(s["qr"], s["kr"], s["vt"], p["log_decay"], lengths=lengths,
                                                return_state=True)
    s["ot"] = s["out"].transpose(1, 2)
    s["o"] = pkg.layer_norm(s["ot"], p["wo"], p["bo"])
    return s


def cpu(d):
    return {n: t.detach().cpu() for n, t in d.items()}


def norm_size(x, eps=1e-5):
    x = x.double()
    r = 1 / torch.sqrt((x - x.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps)
    return r, (x.abs() + x.abs().mean(-1, keepdim=True)) * r


def check_norm(x, w, b, y):
    _, size = norm_size(x)
    within(y, mixer_ref.layer_norm(x, w, b), 2 * size * w.double().abs() + (0 if b is None else b.double().abs()), y.dtype,
           steps(x.shape[-1]))


def check_norm_back(x, w, dy, dx, dw, db):
    r, size = norm_size(x)
    D, rows = x.shape[-1], x.numel() // w.numel()
    wx, wdw, wdb = mixer_ref.layer_norm_backward(dy, x, w)
    gw, h, lead = dy.double().abs() * w.double().abs(), size + 1, tuple(range(x.ndim - w.ndim))
    within(dx, wx, 4 * r * (gw + gw.mean(-1, keepdim=True) + h * (gw * h).mean(-1, keepdim=True)), dx.dtype, steps(D))
    chain = (rows / 512 + 64 + 64 + 64) * 2.0 ** -24
    within(dw, wdw, (dy.double().abs() * size).sum(lead), torch.float32, steps(D) + chain)
    if db is not None:
        within(db, wdb, dy.double().abs().sum(lead), torch.float32, chain)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,N,lengths", [(1, 1, None), (3, 150, [150, 0, 77]), (2, 65, [64, 65])])
def test_layer_forward_and_backward(pkg, device, B, N, lengths, dtype):
    """Training on a padded batch: every stage and every gradient against float64."""
    plan = pkg.rotary_plan(32, device=device)
    p, up = make(B, N, dtype, seed=N)
    p = {n: t.to(device).requires_grad_(True) for n, t in p.items()}
    positions = torch.arange(N, device=device)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    s = layer(pkg, p, positions, plan, ln)
    inner = ("y", "qn", "kn", "qr", "kr", "vt", "out", "q", "k")
    grads = torch.autograd.grad(s["o"], [p[n] for n in PARAMETERS] + [s[n] for n in inner], up.to(device))
    d = cpu(dict(zip([*PARAMETERS, *inner], grads)))
    p, s = cpu(p), cpu(s)
    host_lengths = None if lengths is None else torch.tensor(lengths)
    check_norm(p["x"], p["w"], p["b"], s["y"])
    check_norm(s["q"], p["wq"], None, s["qn"])
    check_norm(s["k"], p["wk"], None, s["kn"])
    check_norm(s["ot"], p["wo"], p["bo"], s["o"])
    f, pos = plan.inverse_frequencies, torch.arange(N)
    for a, b in (("qn", "qr"), ("kn", "kr")):
        x = s[a].transpose(1, 2)
        within(s[b], mixer_ref.rotary(x, pos, f, False), rotary_terms(x, plan), dtype, rotary_slack(dtype))
        u = d[b]
        within(d[a].transpose(1, 2), mixer_ref.rotary(u, pos, f, False, inverse=True), rotary_terms(u, plan), dtype,
               rotary_slack(dtype))
    args = (s["qr"], s["kr"], s["vt"], p["log_decay"], 0.125)
    size = tuple(t.abs() if i < 3 else t for i, t in enumerate(args))
    (want, wstate), (terms, tstate) = (mixer_ref.linear_attention(*a, None, host_lengths) for a in (args, size))
    within(s["out"], want, terms, dtype, attention_slack(dtype))
    within(s["state"], wstate, tstate, torch.float32, FP32)
    wants = mixer_ref.linear_attention_backward(*args, d["out"], None, host_lengths)
    sizes = mixer_ref.linear_attention_backward(*size, d["out"].abs(), None, host_lengths)
    for n, w, t in zip(("qr", "kr", "vt"), wants, sizes):
        within(d[n], w, t, dtype, attention_slack(dtype))
    # as in the operator's own test; no final state's gradient enters
    flow = (size[0].double() * sizes[0]).sum((0, 2, 3))
    within(d["log_decay"], wants[3], 3 * 256 * flow, torch.float32, attention_slack(dtype))
    check_norm_back(s["ot"], p["wo"], up, d["out"].transpose(1, 2), d["wo"], d["bo"])
    check_norm_back(s["q"], p["wq"], d["qn"], d["q"], d["wq"], None)
    check_norm_back(s["k"], p["wk"], d["kn"], d["k"], d["wk"], None)
    check_norm_back(p["x"], p["w"], d["y"], d["x"], d["w"], d["b"])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_prompts_then_single_tokens(pkg, device, dtype):
    """Prompts of several lengths in one padded call, their states in a pool, then tokens one by one, with a row that pads
    the batch: the states and the tokens' outputs are the recurrence's over the whole sequences."""
    B, N, T, P = 3, 130, 6, 8
    lengths, slots = [130, 1, 70], [5, 0, 3]
    plan = pkg.rotary_plan(64, interleaved=True, device=device)
    p = {n: t.to(device) for n, t in make(B, N, dtype, seed=5)[0].items()}
    s = layer(pkg, p, torch.arange(N, device=device), plan, torch.tensor(lengths, device=device))
    pool = torch.full((P, H, HD, HD), 3.0, device=device)
    pool[slots] = s["state"]
    rows = torch.tensor([*slots, -1], device=device)   # the fourth row pads the batch
    at = torch.tensor([[n] for n in [*lengths, 0]], device=device)
    ks, vs, qs, outs = ([] for _ in range(4))
    tokens = make(4, T, dtype, seed=6)[0]["x"].to(device)
    for t in range(T):
        q, k, v = split(pkg.layer_norm(tokens[:, t:t + 1], p["w"], p["b"]))
        q, k = pkg.layer_norm(q, p["wq"]), pkg.layer_norm(k, p["wk"])
        q, k = pkg.rotary_embed(q.transpose(1, 2), k.transpose(1, 2), at + t, plan)
        out = pkg.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, 0], p["log_decay"], pool, slots=rows)
        assert not bool(out[3].any())
        for kept, x in ((qs, q), (ks, k), (vs, v.transpose(1, 2)), (outs, out[:, :, None])):
            kept.append(x.cpu())
    assert bool((pool[[1, 2, 4, 6, 7]] == 3.0).all())
    for b, n in enumerate(lengths):
        whole = [torch.cat([s[name][b:b + 1, :, :n].cpu(), *(x[b:b + 1] for x in kept)], 2)
                 for name, kept in (("qr", qs), ("kr", ks), ("vt", vs))]
        lg = p["log_decay"].cpu()
        want, wstate = mixer_ref.linear_attention(*whole, lg, 0.125)
        terms, tstate = mixer_ref.linear_attention(*(x.abs() for x in whole), lg, 0.125)
        got = torch.cat([x[b:b + 1] for x in outs], 2)
        # the prompt's state, then a decay weight, a product and a sum for each token (50 half steps, as in test_step)
        more = 50 * T * 2.0 ** -24
        within(got, want[:, :, n:], terms[:, :, n:], dtype, FP32 + more)
        within(pool[slots[b]], wstate[0], tstate[0], torch.float32, FP32 + more)


def test_layer_in_graphs_and_on_two_streams(pkg, device):
    """The layer with its gradients captured twice, both graphs replayed in turn with eager work between, and on two
    streams at once: the eager calls' bits every time."""
    plan = pkg.rotary_plan(64, device=device)
    positions, lengths = torch.arange(100, device=device), torch.tensor([100, 31], dtype=torch.int32, device=device)
    sides = []
    for seed in (1, 2):
        p, up = make(2, 100, torch.bfloat16, seed)
        sides.append(({n: t.to(device).requires_grad_(True) for n, t in p.items()}, up.to(device)))

    def work(p, up):
        s = layer(pkg, p, positions, plan, lengths)
        return [s["o"].detach(), s["state"].detach(), *torch.autograd.grad(s["o"], [p[n] for n in PARAMETERS], up)]

    want = [[t.clone() for t in work(*side)] for side in sides]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sides], [None, None]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, side in enumerate(sides):
            with torch.cuda.stream(streams[i]):
                got[i] = work(*side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for side in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(*side))
    base = [side[0]["x"].detach().clone() for side in sides]
    for rep in range(3):
        for i, side in enumerate(sides):
            with torch.no_grad():
                side[0]["x"].copy_(base[i] * (1 + rep))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        kept = [[t.clone() for t in o] for o in outs]
        for i, side in enumerate(sides):
            assert all(torch.equal(x, y) for x, y in zip(kept[i], work(*side))), (rep, i)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_tensors_that_begin_at_odd_addresses(pkg, device, dtype):
    """Dense tensors one element into their memory: the same bits as aligned ones."""
    g = torch.Generator().manual_seed(3)

    def odd(t):
        y = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape)
        return y.copy_(t)

    q, k, v = (randn(g, 2, n, 70, HD, dtype=dtype).to(device) for n in (H, HKV, HKV))
    lg, initial = -torch.rand(H, generator=g).to(device), randn(g, 2, H, HD, HD).to(device)
    plan, pos = pkg.rotary_plan(64, interleaved=True, device=device), torch.arange(70, device=device)
    a = pkg.linear_attention(q, k, v, lg, initial_state=initial, return_state=True)
    b = pkg.linear_attention(odd(q), odd(k), odd(v), odd(lg), initial_state=odd(initial), return_state=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(pkg.rotary_embed(q, k, pos, plan), pkg.rotary_embed(odd(q), odd(k), odd(pos), plan)))
    pools = [initial.clone(), initial.clone()]
    a = pkg.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lg, pools[0])
    b = pkg.linear_attention_step(odd(q[:, :, 0]), odd(k[:, :, 0]), odd(v[:, :, 0]), odd(lg), pools[1])
    assert torch.equal(a, b) and torch.equal(*pools)
    x, w = randn(g, 5, 72, dtype=dtype).to(device), randn(g, 72).to(device)
    want = mixer_ref.layer_norm(x.cpu(), w.cpu())
    _, size = norm_size(x.cpu())
    within(pkg.layer_norm(odd(x), odd(w)), want, 2 * size * w.cpu().double().abs(), dtype, steps(72))


def test_indices_beyond_32_bits(pkg, device):
    """64-bit lengths and slots keep their meaning: above every length, outside every pool."""
    g = torch.Generator().manual_seed(4)
    q, k, v = (randn(g, 5, n, 9, HD).to(device) for n in (H, HKV, HKV))
    lg = -torch.rand(H, generator=g).to(device)
    big = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5, 2 ** 63 - 1, -2 ** 63, 3], device=device)
    small = torch.tensor([9, 0, 9, 0, 3], dtype=torch.int32, device=device)
    a, b = (pkg.linear_attention(q, k, v, lg, lengths=n, return_state=True) for n in (big, small))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    pool = randn(g, 6, H, HD, HD).to(device)
    before = pool.clone()
    out = pkg.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], lg, pool, slots=big)
    assert torch.equal(pool[[0, 1, 2, 4, 5]], before[[0, 1, 2, 4, 5]]) and not torch.equal(pool[3], before[3])
    assert not bool(out[:4].any()) and bool(out[4].any())


def test_more_threads_than_one_dimension_of_a_grid(pkg, device):
    """2^30 + 1,000 rows of one pair, a thread each: the rotary kernel's second dimension."""
    n = (1 << 30) + 1000
    x = torch.randn(1, 1, n, 2, dtype=torch.float16, device=device)
    y, _ = pkg.rotary_embed(x, None, torch.zeros(1, dtype=torch.int32, device=device).expand(n), pkg.rotary_plan(2, device=device))
    assert torch.equal(y, x)
