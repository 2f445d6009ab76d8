"""GPU tests of the mixer's eager calls where something else than a plain launch has to see them: dispatch modes, traces
(make_fx, torch.jit.trace), fake tensors, batched gradients, function transforms, tensors that stand for other values than
their memory holds.  They take the custom ops, so the results are the plain calls' bits.
"""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from tests.mixer_cases import randn

pytestmark = pytest.mark.gpu
H, HKV, N, HD = 4, 2, 100, 64


class Seen(TorchDispatchMode):
    """The names of the operators that the dispatcher sees."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.fixture
def x(pkg, device):
    g = torch.Generator().manual_seed(1)
    heads = lambda n, dtype=torch.bfloat16: randn(g, 2, N, n, HD, dtype=dtype).transpose(1, 2)   # noqa: E731
    t = dict(q=heads(H), k=heads(HKV), v=heads(HKV), log_decay=-torch.rand(H, generator=g) / 8, initial=randn(g, 2, H, HD, HD),
             rows=randn(g, 6, H, HD), weight=1 + 0.2 * randn(g, H, HD), bias=randn(g, H, HD), positions=torch.arange(N) + 3)
    t = {n: v.to(device) for n, v in t.items()}
    t["plan"] = pkg.rotary_plan(32, device=device)
    return t


LEAVES = ("q", "k", "v", "log_decay", "initial", "rows", "weight", "bias")


def calls(pkg, t):
    """The operators' outputs, a stage each."""
    qr, kr = pkg.rotary_embed(t["q"], t["k"], t["positions"], t["plan"])
    out, state = pkg.linear_attention(qr, kr, t["v"], t["log_decay"], initial_state=t["initial"], return_state=True)
    return [qr, kr, out, state, pkg.layer_norm(t["rows"], t["weight"], t["bias"])]


def step(pkg, t, **kw):
    pool = t["initial"].detach().clone()
    with torch.no_grad():
        out = pkg.linear_attention_step(t["q"][:, :, 0], t["k"][:, :, 0], t["v"][:, :, 0], t["log_decay"], pool, **kw)
    return [out, pool]


def leaves_of(t):
    return dict(t, **{n: t[n].detach().clone().requires_grad_(True) for n in LEAVES})


def gradients(pkg, t, ups=None, outs=None):
    outs = calls(pkg, t) if outs is None else outs
    ups = ups or [torch.ones_like(o) for o in outs[2:]]
    return torch.autograd.grad(outs[2:], [t[n] for n in LEAVES], ups)


def same(a, b):
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_dispatch_modes_see_the_operators(pkg, device, x):
    """Forward, forward with gradients, and a backward whose forward ran before the mode."""
    want, want_step = calls(pkg, x), step(pkg, x)
    with Seen() as seen:
        got, got_step = calls(pkg, x), step(pkg, x)
        out = torch.empty_like(want_step[0])
        assert step(pkg, x, out=out)[0] is out
    same(got, want)
    same(got_step, want_step)
    assert torch.equal(out, want_step[0])
    for name, times in (("rotary", 1), ("linear_attention_fwd", 1), ("layer_norm_fwd", 1), ("linear_attention_step_", 2)):
        assert seen.names.count(f"dwarf.{name}.default") == times
    want = gradients(pkg, leaves_of(x))
    with Seen() as seen:
        got = gradients(pkg, leaves_of(x))
    same(got, want)
    t = leaves_of(x)
    outs = calls(pkg, t)
    with Seen() as later:
        same(gradients(pkg, t, outs=outs), want)
    for names in (seen.names, later.names):
        for name in ("rotary", "linear_attention_bwd", "layer_norm_bwd"):
            assert f"dwarf.{name}.default" in names


def test_make_fx_records_calls_and_gradients(pkg, device, x):
    from torch.fx.experimental.proxy_tensor import make_fx

    def work(*leaves):
        t = dict(x, **dict(zip(LEAVES, leaves)))
        outs = calls(pkg, t)
        return [*outs, *gradients(pkg, t, outs=outs), *step(pkg, t)]

    first = [leaves_of(x)[n] for n in LEAVES]
    graph = make_fx(work)(*first)
    names = [str(n.target) for n in graph.graph.nodes]
    for name, times in (("rotary", 2), ("linear_attention_fwd", 1), ("linear_attention_bwd", 1), ("layer_norm_fwd", 1),
                        ("layer_norm_bwd", 1), ("linear_attention_step_", 1)):
        assert names.count(f"dwarf.{name}.default") == times, name
    other = [(t.detach() * 0.5).requires_grad_(True) for t in first]   # the graph on other values
    same(graph(*other), work(*other))


def test_jit_trace_records_the_operators(pkg, device, x):
    def work(q, k, v, rows):
        t = dict(x, q=q, k=k, v=v, rows=rows)
        return tuple(calls(pkg, t))

    first = tuple(x[n] for n in ("q", "k", "v", "rows"))
    traced = torch.jit.trace(work, first, check_trace=False)
    graph = str(traced.graph)
    for name in ("rotary", "linear_attention_fwd", "layer_norm_fwd"):
        assert f"dwarf::{name}" in graph, name
    other = tuple(t * 0.5 for t in first)
    same(traced(*other), work(*other))


def test_fake_tensors_with_gradients(pkg, device, x):
    """Shapes and types of outputs and gradients, also of a backward whose tensors are fake."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    want = [*calls(pkg, x), *gradients(pkg, leaves_of(x)), *step(pkg, x)]
    with FakeTensorMode() as mode:
        t = {n: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for n, v in x.items()}
        plan = pkg.rotary_plan.__globals__["RotaryPlan"].__new__(type(x["plan"]))
        plan.__dict__.update(x["plan"].__dict__, turns=mode.from_tensor(x["plan"].turns))
        t["plan"] = plan
        got = [*calls(pkg, t), *gradients(pkg, leaves_of(t)), *step(pkg, t)]
    assert all(isinstance(g, FakeTensor) for g in got)
    assert [(g.shape, g.dtype, g.stride()) for g in got] == [(w.shape, w.dtype, w.stride()) for w in want]


def test_negated_and_zero_tensors(pkg, device, x):
    """A tensor whose sign is a bit of its own (torch._neg_view) counts as its value, in calls and in gradients."""
    names = ("q", "k", "v", "initial", "rows", "weight", "bias")
    turned = dict(x, **{n: torch._neg_view(-x[n]) for n in names})
    assert all(turned[n].is_neg() for n in names)
    same(calls(pkg, turned), calls(pkg, x))
    same(step(pkg, turned)[:1], step(pkg, x)[:1])
    t = leaves_of(x)
    outs = calls(pkg, t)
    ups = [torch.randn_like(o) for o in outs[2:]]
    same(gradients(pkg, t, [torch._neg_view(-u) for u in ups], outs), gradients(pkg, t, ups))
    zero = [torch._efficientzerotensor(o.shape, dtype=o.dtype, device=device) for o in outs[2:]]
    t = leaves_of(x)
    got = gradients(pkg, t, zero, calls(pkg, t))
    assert not any(bool(g.any()) for g in got)


def test_batched_gradients_and_transforms(pkg, device, x):
    """Batched output gradients (torch.autograd.grad's is_grads_batched) and torch.func transforms: the loop's values or an
    error, never a launch on a wrapped tensor."""
    t = leaves_of(x)
    outs = calls(pkg, t)
    g = torch.Generator().manual_seed(2)
    many = [torch.stack([randn(g, *o.shape).to(o) for _ in range(3)]) for o in outs[2:]]
    args = (outs[2:], [t[n] for n in LEAVES])
    want = [torch.autograd.grad(*args, [m[i] for m in many], retain_graph=True) for i in range(3)]
    try:
        got = torch.autograd.grad(*args, many, is_grads_batched=True)
    except RuntimeError as e:
        assert "vmap" in str(e) or "batch" in str(e), e
    else:
        same(got, [torch.stack(w) for w in zip(*want)])
    rows = torch.stack([x["rows"], 2 * x["rows"] + 1])
    try:
        got = torch.func.vmap(lambda r: pkg.layer_norm(r, x["weight"], x["bias"]))(rows)
    except RuntimeError as e:
        assert "vmap" in str(e) or "batch" in str(e), e
    else:
        same([got], [torch.stack([pkg.layer_norm(r, x["weight"], x["bias"]) for r in rows])])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda r: pkg.layer_norm(r, x["weight"]).sum())(x["rows"])


def test_forward_mode_derivatives_are_refused(pkg, device, x):
    import torch.autograd.forward_ad as fw
    for name in LEAVES:
        with fw.dual_level():
            t = dict(x, **{name: fw.make_dual(x[name], torch.ones_like(x[name]))})
            with pytest.raises(RuntimeError, match="forward mode"):
                calls(pkg, t)
    t = leaves_of(x)
    outs = calls(pkg, t)
    for i in (2, 3, 4):   # output gradients with tangents: forward mode over the backward
        with fw.dual_level():
            up = torch.ones_like(outs[i])
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(outs[i], [t[n] for n in (LEAVES[:5] if i < 4 else LEAVES[5:])],
                                    fw.make_dual(up, up.clone()), retain_graph=True)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_compiled_step_matches_eager(pkg, device, x, index):
    """linear_attention_step in a compiled call: the pool in place, and from one pool into another."""
    rows = [x[n][:, :, 5] for n in ("q", "k", "v")]
    slots = torch.tensor([3, -1], dtype=index, device=device)
    start = torch.randn(5, H, HD, HD, generator=torch.Generator().manual_seed(3)).to(device)

    def in_place(q, k, v, lg, pool, slots):
        out = pkg.linear_attention_step(q, k, v, lg, pool, slots=slots)
        return out * 2, pool.sum()

    def across(q, k, v, lg, pool, new, slots):
        return pkg.linear_attention_step(q, k, v, lg, pool, slots=slots, new_state=new, scale=0.5)

    compile_ = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True)   # noqa: E731
    results = []
    for f, g in ((in_place, across), (compile_(in_place), compile_(across))):
        pool, old, new = start.clone(), start.clone(), torch.zeros_like(start)
        for _ in range(2):
            a, total = f(*rows, x["log_decay"], pool, slots)
        b = g(*rows, x["log_decay"], old, new, slots)
        results.append([a, total, pool, b, old, new])
    same(*results)
    assert torch.equal(results[0][4], start) and not torch.equal(results[0][2], start)
    with pytest.raises(Exception, match="torch.compile"):
        compile_(lambda o: pkg.linear_attention_step(*rows, x["log_decay"], start, slots=slots, out=o))(torch.empty_like(rows[0]))


def test_results_of_calls_without_gradients_are_tensors_of_their_own(pkg, device, x):
    """What a call under no_grad returns may be changed in place with gradients on, as any operator's result may."""
    with torch.no_grad():
        results = calls(pkg, x)
    gate = torch.full((), 0.5, device=device, requires_grad=True)
    for t in results:
        assert not t._is_view()
        half = t * 0.5
        t.mul_(gate)
        assert t.requires_grad and torch.equal(t.detach(), half)
