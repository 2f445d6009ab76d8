"""GPU tests of layer_norm against float64.

Error bound in fp32 half steps: sums over D in a tree of lanes and a chain in each (the chain below 64 terms for rows in
registers, D / 256 for longer ones), so mean and variance are within 100 + D / 128 of their terms; the variance enters
by half.  The centred value loses the mean's error: relative to |x| and |mean|, not to the difference.
"""

import pytest
import torch

from oracle import mixer_ref
from tests.mixer_cases import DTYPES, HALF_STEP, randn, within

pytestmark = pytest.mark.gpu


def steps(D):
    return (100 + D / 128) * 2.0 ** -24


def make(shape, dtype, seed, groups=1, table=torch.float32, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (offset * randn(g, *shape[:-1], 1) + torch.exp(randn(g, *shape[:-1], 1)) * randn(g, *shape)).to(dtype)
    w = (1 + 0.3 * randn(g, *(shape[-2:] if groups > 1 else shape[-1:]))).to(table)
    return x, w, (0.3 * randn(g, *w.shape)).to(table), randn(g, *shape, dtype=dtype)


def check(pkg, device, x, w, b, dy, eps=1e-5, place=lambda t: t):
    D = x.shape[-1]
    dx, dev = place(x.to(device)), []
    leaves = [dx.requires_grad_(True)]
    for t in (w, b):
        dev.append(None if t is None else t.to(device).requires_grad_(True))
        if t is not None:
            leaves.append(dev[-1])
    y = pkg.layer_norm(dx, *dev, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    want = mixer_ref.layer_norm(x, w, b, eps)
    xd = x.double()
    var = (xd - xd.mean(-1, keepdim=True)).square().mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    ww = torch.ones((), dtype=torch.float64) if w is None else w.double().abs()
    # (x - mean) r w + b: |x| + mean |x| carries the mean's error
    size = (xd.abs() + xd.abs().mean(-1, keepdim=True)) * r
    within(y, want, size * ww * 2 + (0 if b is None else b.double().abs()), x.dtype, steps(D))
    got = torch.autograd.grad(y, leaves, place(dy.to(device)))
    wx, wdw, wdb = mixer_ref.layer_norm_backward(dy, x, w, eps)
    gw = dy.double().abs() * ww
    h = size + 1
    terms = r * (gw + gw.mean(-1, keepdim=True) + h * (gw * h).mean(-1, keepdim=True))
    within(got[0], wx, 4 * terms, x.dtype, steps(D))
    rest = list(got[1:])
    lead = tuple(range(x.ndim - (1 if (w if w is not None else b) is None else (w if w is not None else b).ndim)))
    rows = x.numel() // D
    # rows of a thread in a chain (at most rows / 512 + 64), then up to 64 rows of a workgroup and 512 partials
    chain = (rows / 512 + 64 + 64 + 64) * 2.0 ** -24
    if w is not None:
        d = rest.pop(0)
        assert d.dtype == w.dtype and d.shape == w.shape
        within(d, wdw, (dy.double().abs() * size).sum(lead), w.dtype, steps(D) + chain)
    if b is not None:
        d = rest.pop(0)
        assert d.dtype == b.dtype and d.shape == b.shape
        within(d, wdb if w is not None else dy.double().sum(lead), dy.double().abs().sum(lead), b.dtype, chain)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [2051, 8184, 16384, 16392, 20001])
def test_longest_rows(pkg, device, dtype, D):
    """The last widths that registers hold, with and without vectors, and rows that are streamed."""
    check(pkg, device, *make((3, 5, D), dtype, seed=D))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [1, 2, 7, 8, 63, 64, 65, 100, 256, 512, 513, 1024, 1031, 1536, 2056, 4096, 8200])
def test_widths(pkg, device, dtype, D):
    check(pkg, device, *make((5, 7, D), dtype, seed=D))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 16384), (torch.bfloat16, 16392), (torch.bfloat16, 20001),
                                     (torch.float32, 8196), (torch.float32, 20000)])
def test_long_rows(pkg, device, dtype, D):
    check(pkg, device, *make((70, D), dtype, seed=D))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("G,D", [(2, 64), (8, 64), (3, 64), (5, 40), (100, 64), (7, 65), (33, 8), (2, 600), (3, 9000)])
def test_groups(pkg, device, dtype, G, D):
    check(pkg, device, *make((3, 11, G, D), dtype, seed=G * D, groups=G))


@pytest.mark.parametrize("rows", [1, 63, 1000, 5000])
def test_row_counts_and_table_types(pkg, device, rows):
    check(pkg, device, *make((rows, 8, 64), torch.bfloat16, seed=rows, groups=8, table=torch.bfloat16))
    check(pkg, device, *make((rows, 512), torch.bfloat16, seed=rows))


def test_without_weight_or_bias(pkg, device):
    x, w, b, dy = make((33, 96), torch.bfloat16, seed=1)
    check(pkg, device, x, None, None, dy)
    check(pkg, device, x, w, None, dy)
    check(pkg, device, x, None, b, dy)


def test_strided_inputs(pkg, device):
    """A slice of a wider projection, head-major heads, rows off 16-byte alignment: the bits of the contiguous call."""
    x, w, b, dy = make((2, 30, 4, 64), torch.bfloat16, seed=2, groups=4)

    def wide(t):
        base = torch.zeros(*t.shape[:2], 3, *t.shape[2:], device=t.device, dtype=t.dtype)
        base[:, :, 1] = t.detach()
        return base[:, :, 1].detach()

    def headed(t):
        return t.detach().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)

    def shifted(t):
        base = torch.zeros(*t.shape[:-1], 67, device=t.device, dtype=t.dtype)[..., 1:65]
        return base.copy_(t.detach()).detach()

    for place in (wide, headed, shifted):
        check(pkg, device, x, w, b, dy, place=place)
    base = pkg.layer_norm(x.to(device), w.to(device), b.to(device))
    for place in (wide, headed):
        assert torch.equal(pkg.layer_norm(place(x.to(device)), w.to(device), b.to(device)), base)


def test_rows_far_off_centre(pkg, device):
    """Mean 1000 times the spread: the two passes keep the variance to the rounding of x - mean."""
    g = torch.Generator().manual_seed(3)
    x = 1000.0 + randn(g, 20, 300)
    y = pkg.layer_norm(x.to(device)).double().cpu()
    # the mean is off by half a step of 1000 (2^-15) and a few of its sum's, against a spread of 1
    assert float((y - mixer_ref.layer_norm(x)).abs().max()) <= 16 * 2.0 ** -24 * 1000 * 4


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_one_value_have_no_gradient(pkg, device, dtype):
    """y is the bias whatever x holds: dx and dw are 0 themselves."""
    g = torch.Generator().manual_seed(5)
    x, dy = (torch.randn(1000, 1, generator=g).to(dtype).to(device) for _ in range(2))
    w, b = (torch.randn(1, generator=g).to(device) for _ in range(2))
    for t in (x, w, b):
        t.requires_grad_(True)
    y = pkg.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(y, b.to(dtype).expand_as(y)) and not dx.any() and not dw.any() and db.any()


def test_constant_rows_and_values_that_are_not_numbers(pkg, device):
    """A constant row gives the bias; a NaN or infinity spoils its own row alone."""
    x = torch.full((6, 130), 3.0)
    x[4, 7], x[5, 8] = float("nan"), float("inf")
    b = torch.linspace(-1, 1, 130)
    y = pkg.layer_norm(x.to(device), None, b.to(device)).cpu()
    assert torch.equal(y[:4], b.expand(4, 130))
    assert bool(y[4:].isnan().all())


def test_empty_rows(pkg, device):
    x = torch.empty(0, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    y = pkg.layer_norm(x, w, w.detach())
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_differences(pkg, device):
    """Gradients against central differences of the fp32 kernel, summed in float64."""
    x, w, b, dy = (t.to(device) for t in make((9, 3, 70), torch.float32, seed=5, groups=3))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def loss(t):
        return (pkg.layer_norm(*t, eps=1e-2).double() * dy.double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    g = torch.Generator().manual_seed(6)
    for i, grad in enumerate(grads):
        way = randn(g, *leaves[i].shape).to(device)
        # x: an unevenness of third order, h^2 / 6 of the third derivative (64-bit differences of the oracle give it);
        # w and b: linear
        h = 2.0 ** -6
        with torch.no_grad():
            up, down = (loss([t + s * h * way if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        def ref(s):
            t = [v.cpu().double() for v in (x, w, b)]
            t[i] = t[i] + s * way.cpu().double()
            return float((mixer_ref.layer_norm(*t, eps=1e-2) * dy.cpu().double()).sum())
        third = abs((ref(2 * h) - 2 * ref(h) + 2 * ref(-h) - ref(-2 * h)) / (2 * h ** 3))
        size = float((dy.double().abs() * 8).sum())
        bound = h * h / 6 * third * 2 + steps(70) * size / h
        assert abs(float((up - down) / (2 * h) - (grad.double() * way.double()).sum())) <= bound, i


def test_same_bits_graph_and_compile(pkg, device):
    x, w, b, dy = (t.to(device) for t in make((700, 8, 64), torch.bfloat16, seed=7, groups=8))

    def step(x, w, b):
        return (pkg.layer_norm(x, w, b).float() * dy.float()).sum()

    results = []
    for fn in (step, step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        loss = fn(*leaves)
        loss.backward()
        results.append([loss.detach(), *(t.grad for t in leaves)])
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))

    def raw():
        return [pkg.norm.norm_forward(x, w, b, 8, 1e-5), *pkg.norm.norm_backward(dy, x, w, 8, 1e-5, True, True, True)]

    raw()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = raw()
    for rep in range(3):
        x.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(p, q) for p, q in zip(got, raw())), rep
        torch.cuda.synchronize()
    leaf = x.clone().requires_grad_(True)
    up = dy.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(pkg.layer_norm(leaf, w, b), leaf, up, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().sum(), up)
