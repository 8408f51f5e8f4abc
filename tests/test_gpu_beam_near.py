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


def _row_between(v, score, off, g):
    """fp32 logits whose best value lies `off` above the middle of two neighbouring 64-bit numbers, beside
    `score`: some logits are tuned, each leaves what a step of it is worth."""
    x = (torch.randn(v, generator=g) * 2).numpy()
    x[7] = 12.0
    step = np.spacing(abs(score))
    total = lambda: np.exp(x.astype(np.float64) - 12).sum()  # noqa: E731
    want = np.exp(-((np.floor(-np.log(total()) / step) - 0.5) * step + off))
    for j in range(20, 60):
        rest = want - total() + np.exp(float(x[j]) - 12)
        if rest > 0:
            x[j] = min(12 + np.log(rest), 11.0)
    assert abs(np.log(want / total())) < 1e-11
    return torch.from_numpy(x)


@pytest.mark.parametrize("exponent", [35, 40, 44])
def test_rounding_beside_a_large_score_takes_no_part(exponent):
    """Beams alike, each at its own alignment: their first sums differ by 1e-10 and more, which a rounding to
    2^-17 and more may turn into a step of it.  Equal rows have equal values, whichever side they fall to."""
    g = torch.Generator().manual_seed(exponent)
    score = -2.0 ** exponent
    rows = torch.stack([_row_between(1001, score, off, g) for off in np.linspace(-4e-8, 4e-8, 801)])
    x = rows[:, None].expand(-1, 6, -1).contiguous().to(DEV)
    got = beam_select(x, torch.full((801, 6), score, device=DEV))
    assert (got.tokens == 7).all()
    first = torch.arange(801, device=DEV)[:, None] * 6
    assert torch.equal(got.parents - first, torch.arange(6, device=DEV).expand(801, 6))
