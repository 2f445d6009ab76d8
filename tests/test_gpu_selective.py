"""GPU tests of the selective mixer's operators together, as a block runs them: RMS norm of the residual stream's sum, a
short causal convolution, the selective scan whose step, B, C and gate come from the same row; trained in one call and
served as a prompt and single tokens.  Then the eager calls where something else than a plain launch has to see them.

Each stage is compared with its float64 oracle on the values that reached it (the checks of the operators' own tests), and
the block's values and gradients are the stages' bits.
"""

import threading

import pytest
import torch

from oracle import selective_ref
from tests import test_gpu_conv as conv
from tests import test_gpu_rms as rms
from tests import test_gpu_selscan as scan
from tests.mixer_cases import DTYPES, randn
from tests.selective_cases import U, f64, scan_bounds, silu_off, within
from tests.test_gpu_mixer_traced import Seen

pytestmark = pytest.mark.gpu
D, S, W = 40, 16, 4
CUTS = [D, D, S, S, D]   # the convolution's rows, delta, B, C, gate
WIDTH = sum(CUTS)
PARAMETERS = ("x", "r", "w", "wc", "bc", "A", "skip", "bias", "front", "initial")


def make(B, N, dtype, seed, device="cpu", grad=False):
    g = torch.Generator().manual_seed(seed)
    p = dict(x=randn(g, B, N, WIDTH, dtype=dtype), r=randn(g, B, N, WIDTH), w=1 + 0.2 * randn(g, WIDTH), wc=randn(g, D, W) / 2,
             bc=randn(g, D) / 4, A=-torch.exp(0.5 * randn(g, D, S)), skip=randn(g, D), bias=randn(g, D),
             front=randn(g, B, W - 1, D, dtype=dtype), initial=randn(g, B, D, S))
    ups = [randn(g, B, N, D, dtype=dtype), randn(g, B, N, WIDTH), randn(g, B, W - 1, D, dtype=dtype), randn(g, B, D, S)]
    return {k: v.to(device).requires_grad_(grad) for k, v in p.items()}, [u.to(device) for u in ups]


def block(pkg, p, lengths=None):
    s = {}
    s["y"], s["sum"] = pkg.rms_norm(p["x"], p["w"], residual=p["r"])
    s["rows"], s["delta"], s["B"], s["C"], s["gate"] = s["y"].split(CUTS, -1)
    s["xc"], s["front"] = pkg.causal_conv(s["rows"], p["wc"], p["bc"], activation="silu", initial_state=p["front"], lengths=lengths,
                                          return_state=True)
    s["out"], s["state"] = pkg.selective_scan(s["xc"], s["delta"], p["A"], s["B"], s["C"], skip=p["skip"], gate=s["gate"],
                                              delta_bias=p["bias"], softplus=True, initial_state=p["initial"], lengths=lengths,
                                              return_state=True)
    return s


RESULTS = ("out", "sum", "front", "state")


def same(a, b):
    assert len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,N,lengths", [(1, 1, None), (3, 150, [150, 0, 77]), (2, 65, [64, 65])])
def test_block_forward_and_backward(pkg, device, B, N, lengths, dtype):
    p, ups = make(B, N, dtype, N, device, True)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    s = block(pkg, p, ln)
    inner = ("y", "xc")
    d = dict(zip([*PARAMETERS, *inner], torch.autograd.grad([s[k] for k in RESULTS], [p[k] for k in PARAMETERS] + [s[k] for k in inner],
                                                            ups)))
    leaf = lambda t: t.detach().requires_grad_(True)   # noqa: E731
    c = dict(x=leaf(s["xc"]), delta=leaf(s["delta"]), A=p["A"], B=leaf(s["B"]), C=leaf(s["C"]), skip=p["skip"], gate=leaf(s["gate"]),
             delta_bias=p["bias"], initial=p["initial"], softplus=True, lengths=ln, dy=ups[0], dstate=ups[3])
    out, g = scan.check(pkg, c)
    same([out["y"], out["state"], *(g[k] for k in ("x", "A", "skip", "delta_bias", "initial"))],
         [s["out"], s["state"], d["xc"], d["A"], d["skip"], d["bias"], d["initial"]])
    c = dict(x=leaf(s["rows"]), weight=p["wc"], bias=p["bc"], initial=p["front"], lengths=ln, dy=d["xc"], dstate=ups[2])
    h = conv.check(pkg, c, "silu")
    same([h["weight"], h["bias"], h["initial"]], [d["wc"], d["bc"], d["front"]])
    assert torch.equal(torch.cat([h["x"], g["delta"], g["B"], g["C"], g["gate"]], -1), d["y"])
    rms.check_forward(p["x"].detach(), p["w"], p["r"].detach(), (s["y"], s["sum"]), 1e-5)
    rms.check_backward(p["x"].detach(), p["w"], p["r"].detach(), d["y"], ups[1], 1e-5, [d["x"], d["r"], d["w"]])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_prompts_then_single_tokens(pkg, device, dtype):
    """Prompts of several lengths in one padded call, their states in pools, then tokens one by one, with a row that pads
    the batch: the values of the operators over the whole sequences."""
    B, N, T, P = 3, 130, 6, 8
    lengths, slots = [130, 2, 70], [5, 0, 3]
    p, _ = make(B, N, dtype, 5, device)
    tail = {k: v[:, :T] for k, v in make(4, T, dtype, 6, device)[0].items() if k in ("x", "r")}
    with torch.no_grad():
        s = block(pkg, p, torch.tensor(lengths, device=device))
        fronts = torch.full((P, W - 1, D), 3.0, dtype=dtype, device=device)
        pool = torch.full((P, D, S), 3.0, device=device)
        fronts[slots], pool[slots] = s["front"], s["state"]
        rows = torch.tensor([*slots, -1], device=device)
        kept = {k: [] for k in ("rows", "delta", "B", "C", "gate", "xc", "out")}
        for t in range(T):
            y, _ = pkg.rms_norm(tail["x"][:, t], p["w"], residual=tail["r"][:, t])
            q = dict(zip(("rows", "delta", "B", "C", "gate"), y.split(CUTS, -1)))
            q["xc"] = pkg.causal_conv_step(q["rows"], p["wc"], p["bc"], fronts, activation="silu", slots=rows)
            q["out"] = pkg.selective_scan_step(q["xc"], q["delta"], p["A"], q["B"], q["C"], pool, skip=p["skip"], gate=q["gate"],
                                               delta_bias=p["bias"], softplus=True, slots=rows)
            assert not bool(q["out"][3].any()) and not bool(q["xc"][3].any())
            for k in kept:
                kept[k].append(q[k])
    assert bool((pool[[1, 2, 4, 6, 7]] == 3.0).all()) and bool((fronts[[1, 2, 4, 6, 7]] == 3.0).all())
    for b, n in enumerate(lengths):
        whole = {k: torch.cat([s[k][b:b + 1, :n], torch.stack(v, 1)[b:b + 1]], 1) for k, v in kept.items()}
        w = {k: f64(v) for k, v in whole.items()}
        # one more rounding of the convolution's state than none: its rows are the inputs themselves
        args = (w["rows"], f64(p["wc"]), f64(p["bc"]))
        pre, front = selective_ref.causal_conv(*args, None, f64(p["front"][b:b + 1]))
        size, _ = selective_ref.causal_conv(*(a.abs() for a in args), None, f64(p["front"][b:b + 1]).abs())
        within(whole["xc"], selective_ref.silu(pre), silu_off(pre, (W + 1) * size), dtype, U)
        assert torch.equal(f64(fronts[slots[b]]), front[0])
        ref = dict(x=w["xc"], delta=w["delta"], A=f64(p["A"]), B=w["B"], C=w["C"], skip=f64(p["skip"]), gate=w["gate"],
                   delta_bias=f64(p["bias"]), initial=f64(p["initial"][b:b + 1]))
        want, state = selective_ref.selective_scan(**ref, softplus=True)
        # the prompt was one of a batch: its segments' joins, whose bound a batch of one has at least
        off = scan_bounds(ref, True)
        within(whole["out"], want, off["y"], dtype, U)
        within(pool[slots[b]], state[0], off["state"][0], torch.float32, U)


def test_block_in_graphs_on_two_streams_and_in_threads(pkg, device):
    """The block with its gradients captured twice, both graphs replayed in turn with eager work between, on two streams at
    once, and from two threads: the eager calls' bits every time."""
    lengths = torch.tensor([100, 31], dtype=torch.int32, device=device)
    sides = [make(2, 100, torch.bfloat16, seed, device, True) for seed in (1, 2)]

    def work(p, ups):
        s = block(pkg, p, lengths)
        return [*(s[k].detach() for k in RESULTS), *torch.autograd.grad([s[k] for k in RESULTS], [p[k] for k in PARAMETERS], ups)]

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
        same(a, b)
    results = [[], []]

    def loop(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                results[i] = work(*sides[i])

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(results, want):
        same(a, b)
    del got, results
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
            same(kept[i], work(*side))
        torch.cuda.synchronize()


def test_steps_in_a_graph(pkg, device):
    """A captured token of the whole block, its pools updated in place by every replay."""
    p, _ = make(6, 1, torch.bfloat16, 3, device)
    slots = torch.tensor([4, 1, -1, 0, 4, 2], dtype=torch.int32, device=device)
    start = [torch.randn(5, W - 1, D, device=device).bfloat16(), torch.randn(5, D, S, device=device)]

    def token(fronts, pool):
        with torch.no_grad():
            y, s = pkg.rms_norm(p["x"][:, 0], p["w"], residual=p["r"][:, 0])
            rows, delta, B, C, gate = y.split(CUTS, -1)
            xc = pkg.causal_conv_step(rows, p["wc"], p["bc"], fronts, activation="silu", slots=slots)
            return [s, pkg.selective_scan_step(xc, delta, p["A"], B, C, pool, skip=p["skip"], gate=gate, delta_bias=p["bias"],
                                               softplus=True, slots=slots)]

    token(*(t.clone() for t in start))
    pools, others = [t.clone() for t in start], [t.clone() for t in start]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = token(*pools)
    for rep in range(4):
        p["x"].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        same([*outs, *pools], [*token(*others), *others])


def traced_case(device):
    p, ups = make(2, 70, torch.bfloat16, 9, device)
    return p, ups


def calls(pkg, p):
    s = block(pkg, p)
    return [s[k] for k in RESULTS]


def leaves_of(p):
    return {k: v.detach().clone().requires_grad_(True) for k, v in p.items()}


def gradients(pkg, p, ups, outs=None):
    return torch.autograd.grad(calls(pkg, p) if outs is None else outs, [p[k] for k in PARAMETERS], ups)


def one_token(pkg, p):
    fronts, pool = p["front"].detach().clone(), p["initial"].detach().clone()
    with torch.no_grad():
        q, scale, s = pkg.rms_norm_fp8(p["x"], p["w"], residual=p["r"])
        rows, delta, B, C, gate = p["x"][:, 3].split(CUTS, -1)
        xc = pkg.causal_conv_step(rows, p["wc"], p["bc"], fronts, activation="silu")
        out = pkg.selective_scan_step(xc, delta, p["A"], B, C, pool, skip=p["skip"], gate=gate, delta_bias=p["bias"], softplus=True)
    return [q.view(torch.uint8), scale, s, xc, out, fronts, pool]


FORWARD = ("rms_norm_fwd", "causal_conv_fwd", "selective_scan_fwd")
BACKWARD = ("rms_norm_bwd", "causal_conv_bwd", "selective_scan_bwd")
TOKEN = ("rms_norm_fp8", "causal_conv_step_", "selective_scan_step_")


def test_dispatch_modes_see_the_operators(pkg, device):
    """Forward, forward with gradients, steps, and a backward whose forward ran before the mode."""
    p, ups = traced_case(device)
    want, token = calls(pkg, p), one_token(pkg, p)
    with Seen() as seen:
        got, got_token = calls(pkg, p), one_token(pkg, p)
    same(got, want)
    same(got_token, token)
    assert all(seen.names.count(f"dwarf.{n}.default") == 1 for n in FORWARD + TOKEN)
    want = gradients(pkg, leaves_of(p), ups)
    with Seen() as seen:
        same(gradients(pkg, leaves_of(p), ups), want)
    t = leaves_of(p)
    outs = calls(pkg, t)
    with Seen() as later:
        same(gradients(pkg, t, ups, outs), want)
    assert all(f"dwarf.{n}.default" in names for n in BACKWARD for names in (seen.names, later.names))


def test_make_fx_records_calls_and_gradients(pkg, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    p, ups = traced_case(device)

    def work(*leaves):
        t = dict(zip(PARAMETERS, leaves))
        outs = calls(pkg, t)
        return [*outs, *gradients(pkg, t, ups, outs), *one_token(pkg, t)]

    first = [leaves_of(p)[k] for k in PARAMETERS]
    graph = make_fx(work)(*first)
    names = [str(n.target) for n in graph.graph.nodes]
    assert all(names.count(f"dwarf.{n}.default") == 1 for n in FORWARD + BACKWARD + TOKEN)
    other = [(t.detach() * 0.5).requires_grad_(True) for t in first]
    same(graph(*other), work(*other))


def test_jit_trace_records_the_operators(pkg, device):
    p, _ = traced_case(device)
    work = lambda x, r: tuple(calls(pkg, dict(p, x=x, r=r)))   # noqa: E731
    traced = torch.jit.trace(work, (p["x"], p["r"]), check_trace=False)
    assert all(f"dwarf::{n}" in str(traced.graph) for n in FORWARD)
    other = (p["x"] * 0.5, p["r"] * 2)
    same(traced(*other), work(*other))


def test_fake_tensors_with_gradients(pkg, device):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    p, ups = traced_case(device)
    want = [*calls(pkg, p), *gradients(pkg, leaves_of(p), ups), *one_token(pkg, p)]
    with FakeTensorMode() as mode:
        t, u = {k: mode.from_tensor(v) for k, v in p.items()}, [mode.from_tensor(v) for v in ups]
        got = [*calls(pkg, t), *gradients(pkg, leaves_of(t), u), *one_token(pkg, t)]
    assert all(isinstance(g, FakeTensor) for g in got)
    assert [(g.shape, g.dtype, g.stride()) for g in got] == [(w.shape, w.dtype, w.stride()) for w in want]


def test_compiled_block_with_gradients(pkg, device):
    p, ups = traced_case(device)
    t = leaves_of(p)
    want = [*calls(pkg, t)]
    want = [*(w.detach() for w in want), *gradients(pkg, t, ups, want), *one_token(pkg, p)]
    compile_ = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True)   # noqa: E731
    t = leaves_of(p)
    outs = compile_(lambda *a: calls(pkg, dict(zip(PARAMETERS, a))))(*(t[k] for k in PARAMETERS))
    same([*outs, *gradients(pkg, t, ups, outs), *compile_(lambda *a: one_token(pkg, dict(zip(PARAMETERS, a))))(*(p[k] for k in PARAMETERS))],
         want)


def test_compiled_with_dynamic_shapes(pkg, device):
    """One trace for several sizes and numbers: sizes, eps and scale are symbols there.  The checks still refuse."""
    compile_ = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=True)   # noqa: E731
    whole = compile_(lambda *a: calls(pkg, dict(zip(PARAMETERS, a))))
    token = compile_(lambda *a: one_token(pkg, dict(zip(PARAMETERS, a))))
    for n in (70, 131):
        p, ups = make(2, n, torch.bfloat16, n, device)
        t = leaves_of(p)
        want = [*calls(pkg, t)]
        want = [*(w.detach() for w in want), *gradients(pkg, t, ups, want), *one_token(pkg, p)]
        t = leaves_of(p)
        outs = whole(*(t[k] for k in PARAMETERS))
        same([*outs, *gradients(pkg, t, ups, outs), *token(*(p[k] for k in PARAMETERS))], want)
    norms = compile_(lambda x, w, eps: [pkg.rms_norm(x, w, eps=eps), *pkg.rms_norm(x, w, residual=x, eps=eps), pkg.layer_norm(x, w, eps=eps)])
    heads = compile_(lambda q, d, scale: pkg.linear_attention(q, q, q, d, scale=scale))
    decay = torch.tensor([-0.1, -0.02], device=device)
    for n, number in ((5, 1e-5), (5, 1e-2), (9, 0.5)):
        x, w, q = torch.randn(n, 48, device=device), torch.randn(48, device=device), torch.randn(1, 2, 30 * n, 64, device=device)
        same(norms(x, w, number), [pkg.rms_norm(x, w, eps=number), *pkg.rms_norm(x, w, residual=x, eps=number), pkg.layer_norm(x, w, eps=number)])
        same([heads(q, decay, number)], [pkg.linear_attention(q, q, q, decay, scale=number)])
    for bad in (-1.0, float("inf"), float("nan")):
        with pytest.raises(Exception, match="eps"):
            norms(x, w, bad)
        if bad != -1.0:
            with pytest.raises(Exception, match="scale"):
                heads(q, decay, bad)


def test_negated_and_zero_tensors(pkg, device):
    p, ups = traced_case(device)
    turned = {k: torch._neg_view(-v) for k, v in p.items()}
    same(calls(pkg, turned), calls(pkg, p))
    same(one_token(pkg, turned)[:5], one_token(pkg, p)[:5])
    t = leaves_of(p)
    outs = calls(pkg, t)
    want = torch.autograd.grad(outs, [t[k] for k in PARAMETERS], ups, retain_graph=True)
    same(torch.autograd.grad(outs, [t[k] for k in PARAMETERS], [torch._neg_view(-u) for u in ups], retain_graph=True), want)
    zero = [torch._efficientzerotensor(o.shape, dtype=o.dtype, device=device) for o in outs]
    assert not any(bool(g.any()) for g in torch.autograd.grad(outs, [t[k] for k in PARAMETERS], zero))


def test_batched_gradients(pkg, device):
    """Batched output gradients: the loop's values or an error, never a launch on a wrapped tensor."""
    p, ups = traced_case(device)
    t = leaves_of(p)
    outs = calls(pkg, t)
    many = [torch.stack([u, 2 * u]) for u in ups]
    args = (outs, [t[k] for k in PARAMETERS])
    want = [torch.autograd.grad(*args, [m[i] for m in many], retain_graph=True) for i in range(2)]
    try:
        got = torch.autograd.grad(*args, many, is_grads_batched=True)
    except RuntimeError as e:
        assert "vmap" in str(e) or "batch" in str(e), e
    else:
        same(got, [torch.stack(w) for w in zip(*want)])


def test_pools_count_as_written(pkg, device):
    """A graph that saved a pool notices that a step has written it."""
    p, _ = traced_case(device)
    pool = p["initial"].clone()
    gate = torch.ones((), device=device, requires_grad=True)
    y = (pool * gate).sum()
    rows, delta, B, C, _ = p["x"][:, 3].split(CUTS, -1)
    with torch.no_grad():
        pkg.selective_scan_step(rows, delta, p["A"], B, C, pool)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_results_past_32_bits(pkg, device):
    """Results of more than 2^31 elements: one token over and over, whose rows and gradients are the same once the state has
    settled (a decay of e^-8 forgets the way there)."""
    N, D = (1 << 21) + 77, 1040
    g = torch.Generator().manual_seed(11)
    row, up = (randn(g, 1, 1, D, dtype=torch.bfloat16).to(device) for _ in range(2))
    x, dy = row.expand(1, N, D), up.expand(1, N, D)
    y, _ = pkg.rms_norm(x, residual=x)
    assert torch.equal(y[:, -1], y[:, 0])
    q, scale = pkg.rms_norm_fp8(x)
    assert torch.equal(q[:, -1].float(), q[:, 0].float()) and torch.equal(scale[:, -1], scale[:, 0])
    del y, q, scale
    leaf = x.detach().requires_grad_(True)
    y = pkg.causal_conv(leaf, randn(g, D, 4).to(device), activation="silu")
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(y[:, -1], y[:, 100]) and torch.equal(dx[:, -5], dx[:, 100])
    del y, dx
    one = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=device).expand(1, N, 1)
    y, state = pkg.selective_scan(leaf, one.expand(1, N, D), torch.full((D, 1), -8.0, device=device), one, one, return_state=True)
    dx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(y[:, -1], y[:, 100]) and torch.equal(state[0, :, 0].bfloat16(), y[0, -1])
    assert torch.equal(dx[:, -100], dx[:, 100])


def test_inputs_changed_before_the_backward_are_noticed(pkg, device):
    p, _ = traced_case(device)
    for change_rows in (True, False):
        t, lengths = leaves_of(p), torch.tensor([70, 3], dtype=torch.int32, device=device)
        rows = t["x"][..., :D] * 1
        y = pkg.causal_conv(rows, t["wc"], lengths=lengths)
        (rows if change_rows else lengths).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_compiled_norm_with_one_type(pkg, device):
    """One gradient serves x and the residual in an eager call; a compiled one has two."""
    x, r = (torch.randn(5, 64, device=device).bfloat16().requires_grad_(True) for _ in range(2))
    up = [torch.randn(5, 64, device=device).bfloat16() for _ in range(2)]
    want = torch.autograd.grad(pkg.rms_norm(x, residual=r), [x, r], up)
    out = torch.compile(lambda x, r: pkg.rms_norm(x, residual=r), backend="aot_eager", fullgraph=True)(x, r)
    same(torch.autograd.grad(out, [x, r], up), want)
