"""Continuations whose values are equal in 64 bits though their logits are not: scores beside which logits
vanish, logits whose differences vanish beside the row's largest.  They come by rising beam, those of one
beam by falling logit."""

import math

import numpy as np
import pytest
import torch

import beam_plain as P
from ojasx_amd import beam_select

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
LOWEST = torch.finfo(torch.float32).min


def _check(x, scores, num, finished=None, pad=0):
    got = beam_select(x, scores, num, finished=finished, pad_id=pad)
    logits = x.float().cpu().numpy()
    v = P.values(logits, scores.cpu().numpy(), None if finished is None else finished.cpu().numpy(), pad)
    g, k, n = v.shape
    at = np.arange(k * n)
    for i in range(g):
        value, logit = v[i].reshape(-1), logits[i].reshape(-1)
        possible = value > -np.inf
        order = np.lexsort((at, np.where(possible, -logit, 0), at // n, -value))[:num]
        assert got.parents[i].tolist() == (order // n + k * i).tolist()
        assert got.tokens[i].tolist() == (order % n).tolist()
        with np.errstate(over="ignore"):
            np.testing.assert_allclose(got.scores[i].cpu().numpy(), value[order].astype(np.float32),
                                       rtol=2.0 ** -23, atol=2.0 ** -19)
    return got


def test_three_logits_beside_a_large_score():
    x = torch.tensor([1.0, 2.0, 3.0], device=DEV).reshape(1, 1, 3)
    for score in (-1e30, LOWEST, 1e30):
        assert _check(x, torch.full((1, 1), score, device=DEV), 3).tokens.tolist() == [[2, 1, 0]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("score", [-1e9, -1e17, -1e30, LOWEST])
@pytest.mark.parametrize("k,v,num", [(4, 1001, 8), (3, 5, 15), (8, 50021, 20), (64, 333, 64)])
def test_beams_kept_back_by_a_low_score(dtype, score, k, v, num):
    """One beam that counts, the others at a score from which nothing comes back; groups of those alone."""
    g = torch.Generator().manual_seed(v)
    x = (torch.randn(4, k, v, generator=g) * 3).to(dtype)
    x[2, :, 7:] = -math.inf                        # fewer than asked for in the beam that counts
    x[3, :, ::2] = -math.inf
    scores = torch.full((4, k), score)
    scores[:3, k // 2] = -0.5
    done = torch.zeros(4, k, dtype=torch.bool)
    done[1, 0] = done[2, k - 1] = True
    x, scores, done = x.to(DEV), scores.to(DEV), done.to(DEV)
    _check(x, scores, num)
    _check(x, scores, num, done, 2)


@pytest.mark.parametrize("beams", [1, 5])
def test_differences_that_vanish_beside_the_largest(beams):
    """A few logits far over the others, which differ by less than 64 bits hold beside them."""
    g = torch.Generator().manual_seed(beams)
    x = torch.randn(2, beams, 4000, generator=g) * 1e-30
    for i, at in enumerate((5, 17, 3999)):
        x[:, :, at] = 16 + i
    got = _check(x.to(DEV), torch.zeros(2, beams, device=DEV), 60)
    assert got.tokens[0, :1].tolist() == [3999]
