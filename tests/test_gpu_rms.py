"""GPU tests of rms_norm and rms_norm_fp8 against the float64 formula.

Bounds, in u = 2^-24 (half a step of fp32).  A row's sum of squares is a chain of at most max(32, D / 256) fused steps in a
thread and at most 6 + 8 additions over threads and waves; all its terms are positive, so it is that many u off, relative.
The quotient, eps, square root and reciprocal add 2.5, the square root halves what is in front of it; two products behind it.
``off(D)`` = (max(32, D / 256) + 14) / 2 + 7.  The sum g w s of the backward has the same chain over terms of both signs,
with a product in front and three behind it.  dw adds, behind s r, one step for each row of a thread and of a workgroup and
one for each of its partial rows; both are at most the rows themselves, plus 24 for the last launch's own lanes.
"""

import pytest
import torch

from oracle import selective_ref
from tests.mixer_cases import DTYPES, randn
from tests.selective_cases import U, norm_grid, within

pytestmark = pytest.mark.gpu
STREAMS = [(d, d) for d in DTYPES] + [(d, torch.float32) for d in DTYPES[:2]]


def off(D):
    return ((max(32, D / 256) + 14) / 2 + 7) * U


def check_forward(x, w, residual, got, eps):
    y, s = got if residual is not None else (got, None)
    want, ws = selective_ref.rms_norm(x.cpu(), None if w is None else w.cpu(), None if residual is None else residual.cpu(), eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    if residual is not None:
        assert s.dtype == residual.dtype and torch.equal(s.double().cpu(), ws)
    within(y, want, want.abs(), x.dtype, off(x.shape[-1]))
    return ws


def check_eights(x, w, residual, got, eps):
    q, scale = got[:2]
    want, ws = selective_ref.rms_norm(x.cpu(), None if w is None else w.cpu(), None if residual is None else residual.cpu(), eps)
    if residual is not None:
        assert torch.equal(got[2].double().cpu(), ws)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32 and scale.shape == (*x.shape[:-1], 1)
    top = (want.abs().amax(-1, keepdim=True) / 448).clamp(min=torch.finfo(torch.float32).tiny)
    sc = scale.double().cpu()
    assert bool(((sc - top).abs() <= top * (off(x.shape[-1]) + 2 * U)).all())
    # the quotient's two roundings more; half a step of e4m3, 2^-10 below its normal range
    off_by = off(x.shape[-1]) + 4 * U
    bound = want.abs() * (2.0 ** -4 * (1 + off_by) + off_by) + sc * 2.0 ** -10
    assert bool(((q.double().cpu() * sc - want).abs() <= bound).all())


def check_backward(x, w, residual, dy, dsum, eps, grads):
    s = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    s, dy, wc = s.detach().cpu(), dy.cpu(), None if w is None else w.detach().cpu()
    ds, dw = selective_ref.rms_norm_backward(dy, s, wc, None if dsum is None else dsum.cpu(), eps)
    s, g = s.double(), dy.double().abs()
    D = s.shape[-1]
    r = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    gw = g if wc is None else g * wc.double().abs()
    terms = r * (gw + s.abs() * r * r * (gw * s.abs()).mean(-1, keepdim=True)) + (0 if dsum is None else dsum.cpu().double().abs())
    within(grads[0], ds, terms, x.dtype, 2 * off(D) + max(32, D / 256) * U + 16 * U)
    if residual is not None:
        within(grads[1], ds, terms, residual.dtype, 2 * off(D) + max(32, D / 256) * U + 16 * U)
    if w is not None:
        lead = tuple(range(s.ndim - w.ndim))
        within(grads[-1], dw, (g * s.abs() * r).sum(lead), w.dtype, off(D) + (s.numel() / w.numel() + 26) * U)


def run(pkg, device, shape, dtype, stream=None, wshape=None, wtype=torch.float32, seed=0, eps=1e-5, scale=1.0, use_sum=True):
    g = torch.Generator().manual_seed(seed)
    x = (scale * randn(g, *shape)).to(dtype).to(device).requires_grad_(True)
    w = None if wshape is None else (1 + 0.2 * randn(g, *wshape)).to(wtype).to(device).requires_grad_(True)
    r = None if stream is None else randn(g, *shape, dtype=stream).to(device).requires_grad_(True)
    dy = randn(g, *shape, dtype=dtype).to(device)
    out = pkg.rms_norm(x, w, residual=r, eps=eps)
    check_forward(x.detach(), w, None if r is None else r.detach(), out if r is None else (out[0], out[1]), eps)
    with torch.no_grad():
        check_eights(x, w, r, pkg.rms_norm_fp8(x, w, residual=r, eps=eps), eps)
    leaves = [t for t in (x, r, w) if t is not None]
    dsum = randn(g, *shape, dtype=stream).to(device) if r is not None and use_sum else None
    outs, ups = ([out], [dy]) if r is None else (list(out), [dy, dsum]) if use_sum else ([out[0]], [dy])
    check_backward(x, w, r, dy, dsum, eps, torch.autograd.grad(outs, leaves, ups))


@pytest.mark.parametrize("dtype,stream", STREAMS, ids=str)
@pytest.mark.parametrize("D", [1, 7, 8, 24, 64, 100, 136, 512, 777, 1000, 1024, 2048, 4100, 16384])
def test_widths(pkg, device, dtype, stream, D):
    """Every way a row is shared, in vectors and in single elements, with a residual of both types."""
    run(pkg, device, (9, D), dtype, stream, (D,), seed=D)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("D", [5, 64, 2048, 20000, 33000])
def test_without_residual(pkg, device, dtype, D):
    run(pkg, device, (5, D), dtype, None, (D,), seed=D)
    run(pkg, device, (3, D), dtype, None, None, seed=D + 1)


@pytest.mark.parametrize("dtype,stream", STREAMS, ids=str)
@pytest.mark.parametrize("D", [20000, 33001])
def test_rows_longer_than_the_registers(pkg, device, dtype, stream, D):
    run(pkg, device, (3, 2, D), dtype, stream, (2, D), seed=D)


@pytest.mark.parametrize("G,D", [(1, 64), (3, 40), (5, 7), (32, 64), (7, 1000)])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=str)
def test_groups(pkg, device, dtype, G, D):
    run(pkg, device, (6, 4, G, D), dtype, torch.float32, (G, D), seed=G)


@pytest.mark.parametrize("rows", [1, 63, 64, 65, 3000])
def test_row_counts_and_table_types(pkg, device, rows):
    for wtype in DTYPES:
        run(pkg, device, (rows, 72), torch.bfloat16, torch.bfloat16, (72,), wtype=wtype, seed=rows)
    run(pkg, device, (rows, 72), torch.float16, torch.float32, None, seed=rows, use_sum=False)


@pytest.mark.parametrize("shape,G,dtype,stream", [
    ((9001, 512), 1, torch.bfloat16, torch.bfloat16), ((9001, 512), 1, torch.float16, torch.float32),
    ((30720, 512), 1, torch.bfloat16, torch.float32), ((9001, 512), 1, torch.float32, torch.float32),
    ((24001, 3, 40), 3, torch.bfloat16, torch.float32), ((9500, 8, 64), 8, torch.float16, torch.float16),
    ((9001, 1000), 1, torch.bfloat16, torch.bfloat16), ((9001, 2048), 1, torch.bfloat16, torch.float32),
    ((2500, 1031), 1, torch.float16, torch.float16), ((2500, 8200), 1, torch.bfloat16, torch.float32),
    ((4500, 2000), 1, torch.float32, torch.float32)], ids=str)
def test_more_rows_than_a_grid_holds(pkg, device, shape, G, dtype, stream):
    """Threads that walk over several rows: the bits of calls whose grids hold all their rows.  The weight's gradient adds a
    thread's rows, its workgroup's of the group, and the partial rows, 64 threads to a column and those in five steps, so it is
    a chain of as many steps; each term has s r and the product's rounding."""
    rows, D = shape[0], shape[-1]
    g = torch.Generator().manual_seed(rows + D)
    x, r, dy, ds = (randn(g, *shape, dtype=t).to(device) for t in (dtype, stream, dtype, stream))
    w = (1 + 0.2 * randn(g, *shape[-1 - (G > 1):])).to(device)
    each = 1400 // G
    grids = {back: [norm_grid(n, G, D, dtype, back) for n in (rows, each)] for back in (False, True)}
    assert all(blocks * held < rows * G for blocks, held in (grids[False][0], grids[True][0]))
    assert grids[False][1][0] * grids[False][1][1] >= each * G

    def results(a, b):
        t = [v[a:b].clone().requires_grad_(True) for v in (x, r)] + [w.clone().requires_grad_(True)]
        out = pkg.rms_norm(t[0], t[2], residual=t[1])
        grads = torch.autograd.grad(out, t, [dy[a:b].clone(), ds[a:b].clone()])
        with torch.no_grad():
            q, scale, s = pkg.rms_norm_fp8(t[0], t[2], residual=t[1])
        return [*out, q.view(torch.uint8), scale, s, *grads[:2]], grads[2]

    whole, dw = results(0, rows)
    for a in range(0, rows, each):
        part, _ = results(a, a + each)
        assert all(torch.equal(t[a:a + each], p) for t, p in zip(whole, part)), a
    s, up = whole[1].double(), dy.double()
    terms = up * s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)
    blocks, held = grids[True][0]
    chain = -(-rows * G // (blocks * held)) + -(-held // G) + -(-blocks // 64) + 16 + 2
    off_by = terms.abs().sum(0) * (off(D) + (chain + 2) * U)
    assert bool(((dw.double() - terms.sum(0)).abs() <= off_by + dw.double().abs() * U).all())


@pytest.mark.parametrize("eps,scale", [(0.0, 1.0), (1e-2, 1e-3), (1e-5, 300.0)])
def test_eps_and_sizes(pkg, device, eps, scale):
    run(pkg, device, (8, 200), torch.float16, None, (200,), eps=eps, scale=scale)


def test_only_the_sum_is_used(pkg, device):
    """The stream alone in the loss: its gradient is both inputs', the weight's is zero."""
    g = torch.Generator().manual_seed(1)
    x, w, r, up = (randn(g, *s).to(device).requires_grad_(True) for s in ((4, 48), (48,), (4, 48), (4, 48)))
    _, s = pkg.rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad(s, [x, r, w], up.detach())
    assert torch.equal(dx, up) and torch.equal(dr, up) and not bool(dw.any())


def test_leaves_keep_gradients_of_their_own(pkg, device):
    """x's and the residual's gradients have the same values in memory of their own."""
    x, r = (torch.randn(4, 64, device=device, requires_grad=True) for _ in range(2))
    for _ in range(2):
        y, s = pkg.rms_norm(x, residual=r)
        (y.sum() + (s * s).sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
    before = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, before)


def test_zero_rows_and_values_that_are_not_numbers(pkg, device):
    x = torch.randn(4, 64, device=device).bfloat16()
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    y = pkg.rms_norm(x)
    assert not bool(y[0].any()) and bool(y[1].isnan().all()) and bool(y[2, 5].isnan()) and bool(y[3].isfinite().all())
    q, scale = pkg.rms_norm_fp8(x)
    assert not bool(q[0].float().any()) and float(scale[0]) == torch.finfo(torch.float32).tiny
    assert bool(q[1].float().isnan().all()) and bool(q[2, 5].float().isnan()) and bool(q[3].float().isfinite().all())
    assert torch.equal(y[3], pkg.rms_norm(x[3:4])[0]) and torch.equal(scale[3:], pkg.rms_norm_fp8(x[3:4])[1])


def test_largest_value_of_a_row_is_448(pkg, device):
    """The scale maps a row's largest magnitude on e4m3's largest number, whichever sign it has."""
    x = torch.randn(200, 128, generator=torch.Generator().manual_seed(2)).to(device)
    q, _ = pkg.rms_norm_fp8(x)
    assert torch.equal(q.float().abs().amax(-1), torch.full((200,), 448.0, device=device))


def test_layouts_give_the_same_bits(pkg, device):
    """Strided, expanded, transposed and misaligned inputs against contiguous ones (rows in single elements may add in
    another order, so those are compared with themselves)."""
    g = torch.Generator().manual_seed(3)
    wide = randn(g, 6, 5, 2, 64, dtype=torch.bfloat16).to(device)
    w = randn(g, 2, 64).to(device)
    for x in (wide[:, 1:4], wide.transpose(0, 1), wide[:, :1].expand(6, 5, 2, 64), wide[::2]):
        y, s = pkg.rms_norm(x, w, residual=x)
        cy, cs = pkg.rms_norm(x.contiguous(), w, residual=x.contiguous())
        assert torch.equal(y, cy) and torch.equal(s, cs)
        q, sc = pkg.rms_norm_fp8(x, w)
        cq, csc = pkg.rms_norm_fp8(x.contiguous(), w)
        assert torch.equal(q.view(torch.uint8), cq.view(torch.uint8)) and torch.equal(sc, csc)
    odd = torch.empty(6 * 100 + 1, dtype=torch.bfloat16, device=device)[1:].view(6, 100).normal_(generator=None)
    check_forward(odd, None, None, pkg.rms_norm(odd), 1e-5)
    check_eights(odd, None, None, pkg.rms_norm_fp8(odd), 1e-5)
    ow = torch.empty(101, device=device)[1:].copy_(torch.rand(100, device=device))
    check_forward(odd.clone(), ow, odd.float(), pkg.rms_norm(odd.clone(), ow, residual=odd.float()), 1e-5)
    x = randn(g, 4, 64, 6).to(device).transpose(1, 2)   # elements that do not lie side by side
    assert torch.equal(pkg.rms_norm(x), pkg.rms_norm(x.contiguous()))


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=str)
@pytest.mark.parametrize("D", [64, 512, 2048, 16384])
def test_fp32_streams_at_16_bytes(pkg, device, dtype, D):
    """A stream and its gradient at addresses that 16 divides and 32 does not, as all their rows or as every other one: the
    bits of aligned ones, forward and backward."""
    g = torch.Generator().manual_seed(D)
    x, dy, r, ds = (randn(g, 6, D, dtype=t).to(device) for t in (dtype, dtype, torch.float32, torch.float32))
    w = randn(g, D).to(device)
    want = [*pkg.rms_norm(x, w, residual=r), *(t.view(torch.uint8) if t.element_size() == 1 else t for t in pkg.rms_norm_fp8(x, w, residual=r))]
    back = pkg.norm.rms_backward(dy, ds, r, w, 1, 1e-5, True, True, True)
    for between, start in ((0, 4), (4, 0), (4, 4)):
        def moved(t):
            return torch.empty(6 * (D + between) + start, device=device)[start:].view(6, D + between)[:, :D].copy_(t)
        a, b = moved(r), moved(ds)
        assert a.data_ptr() % 32 == 4 * start and (a.stride(0) * 4) % 32 == 4 * between
        got = [*pkg.rms_norm(x, w, residual=a), *(t.view(torch.uint8) if t.element_size() == 1 else t for t in pkg.rms_norm_fp8(x, w, residual=a))]
        assert all(torch.equal(s, t) for s, t in zip(got, want))
        got = pkg.norm.rms_backward(dy, b, a, w, 1, 1e-5, True, True, True)
        assert all(torch.equal(s, t) for s, t in zip(got, back))


def test_empty_inputs(pkg, device):
    x = torch.empty(0, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    y, s = pkg.rms_norm(x, w, residual=torch.empty(0, 64, device=device))
    assert y.shape == s.shape == (0, 64)
    assert not bool(torch.autograd.grad(y.sum() + s.sum(), w)[0].any())
    with torch.no_grad():
        q, scale = pkg.rms_norm_fp8(x)
    assert q.shape == (0, 64) and scale.shape == (0, 1)


def test_differences(pkg, device):
    """Gradients against central differences in float64, of the function as the formula has it."""
    g = torch.Generator().manual_seed(4)
    x, w, r, a, b = (randn(g, *s) for s in ((3, 20), (20,), (3, 20), (3, 20), (3, 20)))
    leaves = [t.to(device).requires_grad_(True) for t in (x, w, r)]
    y, s = pkg.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    grads = torch.autograd.grad((y * a.to(device)).sum() + (s * b.to(device)).sum(), leaves)

    def f(x, w, r):
        s = x + r
        y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5) * w
        return float((y * a.double()).sum() + (s * b.double()).sum())

    h = 1e-5
    for i, grad in enumerate(grads):
        t = [x.double(), w.double(), r.double()]
        for at in range(0, t[i].numel(), 7):
            d = []
            for sign in (1, -1):
                moved = [v.clone() for v in t]
                moved[i].view(-1)[at] += sign * h
                d.append(f(*moved))
            # the difference's own error: third derivatives h^2 and 2^-53 / h; the gradient's: 1e-5 of terms of size 10
            assert abs((d[0] - d[1]) / (2 * h) - float(grad.reshape(-1)[at])) < 2e-4


def test_far_rows(pkg, device):
    """Rows whose offsets pass 2^31 elements."""
    buf = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device=device)
    x = buf.as_strided((3, 256), ((1 << 30), 1)).normal_()
    assert torch.equal(pkg.rms_norm(x), pkg.rms_norm(x.clone()))


def test_same_bits_graph_and_compile(pkg, device):
    g = torch.Generator().manual_seed(5)
    x, r = (randn(g, 700, 200, dtype=d).to(device).requires_grad_(True) for d in (torch.bfloat16, torch.float32))
    w = randn(g, 200).to(device).requires_grad_(True)
    dy, ds = randn(g, 700, 200, dtype=torch.bfloat16).to(device), randn(g, 700, 200).to(device)

    def work(x, w, r):
        y, s = pkg.rms_norm(x, w, residual=r)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], [x, w, r], [dy, ds])]

    def eights(x, w, r):
        with torch.no_grad():
            q, scale, s = pkg.rms_norm_fp8(x, w, residual=r)
        return [q.view(torch.uint8), scale, s]

    both = lambda: [t.clone() for t in (*work(x, w, r), *eights(x, w, r))]   # noqa: E731
    want = both()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(), want))
    step = torch.compile(lambda x, w, r: pkg.rms_norm(x, w, residual=r), backend="aot_eager", fullgraph=True)
    y, s = step(x, w, r)
    got = [y, s, *torch.autograd.grad([y, s], [x, w, r], [dy, ds])]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.compile(eights, backend="aot_eager", fullgraph=True)(x, w, r)
    assert all(torch.equal(a, b) for a, b in zip(got, want[5:]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    del y, s, got
    with torch.cuda.graph(graph):
        outs = [*work(x, w, r), *eights(x, w, r)]
    for rep in range(3):
        with torch.no_grad():
            x.mul_(1 + rep)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(kept, both())), rep
