"""GPU tests of linear_attention over several long segments (256 to 1,024 tokens, up to eight of them and more), which the
training microbatch, padded prompts and long prompts take.

The segment rule goes by B, H and N alone, so a few live sequences in a batch of empty ones reach every length.
"""

import pytest
import torch

from tests.mixer_cases import DTYPES
from tests.test_gpu_linattn import HD

pytestmark = pytest.mark.gpu


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
