"""GPU tests of linear_attention over several long segments (256 to 1,024 tokens, up to eight of them and more), which the
training microbatch, padded prompts and long prompts take, against the float64 oracle in blocks.

The segment rule goes by B, H and N alone, so a few live sequences in a batch of empty ones reach every length.  Inputs are
positive: nothing cancels, every result is as large as its terms, and a wrong weight in any part of dlog_decay shows.
Bounds: those of test_gpu_linattn.py; dlog_decay adds at most three weights of a segment's tokens times |q.dq|, |k.dk| and
<S, G> at the segments' borders (exact in float64 here), each term formed in fp32: 400 half steps, two more for each
segment that a state has passed.  The results are at least 20 bounds large, so that zeros or half weights cannot pass.
"""

import math

import pytest
import torch

from oracle import mixer_ref
from tests.mixer_cases import DTYPES, within
from tests.test_gpu_linattn import FP32, HD, put, slack

pytestmark = pytest.mark.gpu

CASES = [
    # B, H, Hkv, N, segment, lengths of the live sequences (the others are empty)
    (16, 8, 8, 1600, 512, [1600, 1537, 1090]),          # four segments; tails of 64, 1 and 66 tokens
    (15, 8, 2, 2048, 512, [2048, 1500]),                 # the training microbatch's, shared heads
    (32, 8, 4, 1100, 1024, [1100, 1025]),                # two segments of 1,024, the second with 76 and 1 tokens
    (56, 8, 8, 1088, 1024, [1088, 1030, 1024]),          # two segments of 1,024; tails of 64, 6 and none
    (3, 8, 8, 1300, 128, [1300, 1217]),                  # eleven segments: the scan in groups
    (3, 8, 4, 2600, 256, [2600, 2497, 300]),
    (6, 8, 8, 5200, 512, [5184, 3333]),
    (7, 8, 2, 9300, 1024, [9280, 9000]),                 # ten segments of 1,024, a tail of 64
    (1, 2, 1, 9001, 64, [9001]),                         # 141 segments of one chunk: the scan in two passes
    (1, 2, 2, 16600, 128, [16600]),                      # 130 of two chunks
]


def positive(B, H, Hkv, N, dtype, lengths, seed):
    g = torch.Generator().manual_seed(seed)
    live = len(lengths)

    def heads(n):
        x = torch.zeros(B, N, n, HD, dtype=dtype)
        x[:live] = (torch.rand(live, N, n, HD, generator=g) * 0.9 + 0.1).to(dtype)
        return x.transpose(1, 2)

    x = dict(q=heads(H), k=heads(Hkv), v=heads(Hkv), dout=heads(H))
    x["log_decay"] = torch.log1p(-torch.exp(-torch.linspace(math.log(8.0), math.log(512.0), H)))
    x["initial"], x["dstate"] = torch.rand(B, H, HD, HD, generator=g), torch.rand(B, H, HD, HD, generator=g)
    x["lengths"] = torch.tensor([*lengths] + [0] * (B - live), dtype=torch.int32)
    return x


def check(pkg, device, B, H, Hkv, N, seg, lengths, dtype, enters, leaves, dinitial=True):
    """Forward and gradients of positive inputs; enters, leaves: with a state in front and a gradient of the one behind;
    dinitial: with the gradient of the state that enters."""
    assert pkg.linattn.segment_tokens(B, H, N) == seg
    x = positive(B, H, Hkv, N, dtype, lengths, seed=N)
    if not enters:
        x["initial"] = None
    d = put(x, device)
    names = ["q", "k", "v", "log_decay"] + (["initial"] if enters and dinitial else [])
    for n in names:
        d[n].requires_grad_(True)
    out, state = pkg.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], initial_state=d["initial"], lengths=d["lengths"],
                                      return_state=True)
    outs, ups = ((out, state), (d["dout"], d["dstate"])) if leaves else ((out,), (d["dout"],))
    got = dict(zip(names, torch.autograd.grad(outs, [d[n] for n in names], ups)))
    live = len(lengths)
    rows = {n: None if x[n] is None else x[n][:live] for n in ("q", "k", "v", "dout", "initial", "dstate")}
    want, wstate, grads, crossing = mixer_ref.linear_attention_chunked(
        rows["q"], rows["k"], rows["v"], x["log_decay"], 0.125, rows["dout"], rows["initial"], lengths,
        rows["dstate"] if leaves else None)
    grads = dict(zip(("q", "k", "v", "log_decay", "initial"), grads))
    more = -(-N // seg) * 2 * 2.0 ** -24
    # positive inputs: the results are their terms
    within(out[:live], want, want, dtype, slack(dtype) + more)
    within(state[:live], wstate, wstate, torch.float32, FP32 + more)
    for n in ("q", "k", "v"):
        within(got[n][:live], grads[n], grads[n], dtype, slack(dtype) + more)
    if "initial" in got:
        within(got["initial"][:live], grads["initial"], grads["initial"], torch.float32, FP32 + more)
    # the empty sequences: nothing but the state that goes through
    assert not any(bool(t[live:].any()) for t in (out, got["q"], got["k"], got["v"]))
    assert torch.equal(state[live:], d["initial"][live:]) if enters else not bool(state[live:].any())
    if "initial" in got:
        assert torch.equal(got["initial"][live:], d["dstate"][live:]) if leaves else not bool(got["initial"][live:].any())
    flow = (rows["q"].double() * grads["q"]).sum((0, 2, 3)) + (
        rows["k"].double() * grads["k"]).sum((0, 2, 3)).repeat_interleave(H // Hkv) + sum(
            c for kept in crossing for c in kept[::seg // 64])
    terms = seg * flow
    assert bool((20 * (FP32 + more) * terms < grads["log_decay"]).all())
    within(got["log_decay"], grads["log_decay"], terms, torch.float32, FP32 + more)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,Hkv,N,seg,lengths", CASES)
def test_long_segments(pkg, device, B, H, Hkv, N, seg, lengths, dtype):
    check(pkg, device, B, H, Hkv, N, seg, lengths, dtype, True, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("enters,leaves", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("B,H,Hkv,N,seg,lengths", [
    (57, 8, 8, 1000, 1024, [1000, 70, 64, 1]),           # one segment: with no state on either side there is no scan
    (28, 8, 4, 100, 256, [100, 65, 64]),
    (15, 8, 2, 2048, 512, [2048, 1601, 30]),
    (6, 8, 8, 5200, 512, [5184, 3333])])
def test_segments_with_parts_left_out(pkg, device, B, H, Hkv, N, seg, lengths, dtype, enters, leaves):
    """Without a state that enters, without a gradient of the one that leaves; the entering one needs no gradient."""
    check(pkg, device, B, H, Hkv, N, seg, lengths, dtype, enters, leaves, dinitial=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,H,N,seg", [(57, 8, 1000, 1024), (57, 8, 1088, 1024), (15, 8, 2048, 512), (3, 8, 1300, 128)])
def test_decay_gradients_that_cancel(pkg, device, B, H, N, seg, dtype):
    """Two sequences whose gradients are each other's negative: small whole numbers without a decay (g = 1), whose terms
    are exact in fp32, in another order of the head's elements.  The terms are far beyond 2^24 of their unit, so the sum is 0
    only where it is kept in 64 bits all the way."""
    assert pkg.linattn.segment_tokens(B, H, N) == seg
    g = torch.Generator().manual_seed(N)
    whole = lambda: torch.randint(-3, 4, (H, N, HD), generator=g).float()   # noqa: E731
    q, k, v, dout = whole(), whole(), whole(), whole()
    a, b = torch.randperm(HD, generator=g), torch.randperm(HD, generator=g)

    def batch(x, y):
        t = torch.zeros(B, H, N, HD)
        t[0], t[1] = x, y
        return t.to(device=device, dtype=dtype)

    args = [batch(q, q[..., a]), batch(k, k[..., a]), batch(v, v[..., b])]
    lengths = torch.tensor([N, N] + [0] * (B - 2), dtype=torch.int32, device=device)
    lg = torch.zeros(H, device=device, requires_grad=True)
    out = pkg.linear_attention(*args, lg, lengths=lengths)
    up = batch(dout, -dout[..., b])
    for only, size in ((slice(0, 1), 1e5), (slice(0, 2), None)):
        one = torch.zeros_like(up)
        one[only] = up[only]
        (got,) = torch.autograd.grad(out, lg, one, retain_graph=True)
        if size:   # each by itself is not 0
            assert float(got.abs().min()) > 0 and float(got.abs().max()) > size
        else:
            assert torch.equal(got, torch.zeros_like(got)), got
