"""Alternatives of rows with NaN: it counts as the largest logit, equal ones by rising token."""

import math

import pytest
import torch

import ojasx_amd

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [1, 2, 5, 64, 300, 3000, 40000])
def test_nan_comes_first_wherever_it_is(dtype, v):
    x = torch.randn(8, v, generator=torch.Generator().manual_seed(v)).to(dtype)
    x[0, 0] = math.nan
    x[1] = math.nan
    x[2, [0, v - 1]] = math.nan
    x[3, :] = -math.inf
    x[3, 0] = math.nan
    x[4, v // 2] = math.inf
    x[4, 0] = math.nan
    x[5, 1:] = torch.finfo(dtype).min
    x[5, 0] = -math.nan
    x[6, ::2] = math.nan
    x[7, v // 3:] = math.nan
    top = min(v, 64)
    got = ojasx_amd.token_logprobs(x.to(DEV), torch.zeros(8, dtype=torch.int64, device=DEV),
                                   top_k=top)
    for row, ids in zip(x.tolist(), got.top_ids.tolist()):
        order = sorted(range(v), key=lambda j: (0, 0.0) if math.isnan(row[j]) else (1, -row[j]))
        assert ids == order[:top]
    for t in (got.logprob, got.entropy, got.lse, got.top_logprobs):
        assert t.isnan().all()


@pytest.mark.parametrize("v", [1, 3, 64])
def test_gradient_of_rows_with_nan_and_every_token_an_alternative(v):
    x = torch.randn(2, v, generator=torch.Generator().manual_seed(v)).to(DEV)
    x[0, 0] = math.nan
    x.requires_grad_(True)
    out = ojasx_amd.token_logprobs(x, torch.tensor([0, v - 1], device=DEV), top_k=v)
    assert sorted(out.top_ids[0].tolist()) == sorted(out.top_ids[1].tolist()) == list(range(v))
    g, = torch.autograd.grad(out.logprob.sum() + out.top_logprobs.sum(), [x])
    assert g[0].isnan().all() and torch.isfinite(g[1]).all()
