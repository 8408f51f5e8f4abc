"""Beams whose values are near each other: their sums are formed again in 64 bits."""

import numpy as np
import pytest
import torch

import beam_plain as P
from ojasx_amd import beam_select

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("steps", [1, 2, 3])
@pytest.mark.parametrize("v,num", [(32000, 2), (50021, 1), (1001, 9)])
def test_values_within_two_errors_of_a_sum_are_exact(dtype, steps, v, num):
    """One row under two scores that differ by 2^-20 to 3 * 2^-20 (of 2^-18, what two sums of the first pass
    may be off by).  Values near zero show in fp32 what their sums are off by: 2^-24 of them is all where
    the sums have 64 bits (v terms, 2^-53 each at most: under 2^-37)."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(1, 1, v, generator=g)
    x[0, 0, v // 3] = 6
    x = x.to(dtype).expand(1, 2, v).contiguous()
    row = x[0, 0].double()
    best = row.max() - torch.logsumexp(row, 0)     # -8 to -1: 2^-20 is a whole number of steps
    near = -best.float()
    scores = torch.stack([near, near + steps * 2.0 ** -20]).reshape(1, 2)
    assert (scores[0, 1] - scores[0, 0]).item() == steps * 2.0 ** -20
    got = beam_select(x.to(DEV), scores.to(DEV), num)
    want = P.select(x.float().numpy(), scores.numpy(), num)
    assert np.array_equal(got.parents.cpu().numpy(), want[1])
    assert np.array_equal(got.tokens.cpu().numpy(), want[2])
    first, exact = got.scores.cpu().numpy().astype(np.float64)[0, :2], want[0][0, :2]
    assert (np.abs(first - exact) <= 2.0 ** -24 * np.abs(exact) + 2.0 ** -37).all()
