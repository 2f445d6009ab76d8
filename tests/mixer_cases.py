"""Inputs and error bounds of the mixer's GPU tests."""

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # one rounding, relative
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def within(got, want, terms, dtype, slack):
    """Every element within one rounding to dtype plus ``slack`` of the terms its sum is made of.

    want: float64 result; terms: float64 sum of the absolute values of what is added up."""
    got = got.detach().double().cpu()
    # half a step of the result, also where the computed one is the larger; fp16 and bf16 below their normal range
    # keep an absolute step
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = HALF_STEP[dtype] * (want.abs() + slack * terms) + slack * terms + tiny
    assert bool(torch.isfinite(got).all())
    over = ((got - want).abs() - bound).max()
    assert float(over) <= 0, f"off by {float((got - want).abs().max())}, {float(over)} above the bound"
