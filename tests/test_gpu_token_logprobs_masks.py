"""Rows masked with large finite values, or with a large finite logit.

Bounds: as in the tests of values, an exponent's rounding is its size times 2^-24, that of the
live logits; sums of V terms over at least 64 lanes add (V / 64 + 32) roundings.  A log
probability is rounded to its own size, a log-sum to the row's largest logit.
"""

import numpy as np
import pytest
import torch

import kv8_plain as P
import ojasx_amd
from test_gpu_token_logprobs import DEV, ULP, _check_grad

pytestmark = pytest.mark.gpu


def _rows(v, dtype, far):
    """Logits, masked at random, but for one token, in front, behind; a row of the value alone,
    beside values of twice it, one of its opposite."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(8, v, generator=g)
    x[0, torch.rand(v, generator=g) < 0.9] = far
    x[0, v // 2] = 1.0
    x[1, 1:] = far
    x[2, : v - 2] = far
    x[3, v // 2:] = far
    x[4] = far
    x[5] = far
    x[5, ::3] = 2 * far
    x[6, v // 3] = -far
    x[7, v // 3:v // 3 + 2] = -far
    x[7, torch.rand(v, generator=g) < 0.3] = far
    return x.to(dtype)


FAR = [-1e7, -1e8, -3e8, -1e9, -3e9, -1e10, -1e12, -1e15, -1e20, -1e29, -1e31, -1e37]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [6, 515, 40000])
@pytest.mark.parametrize("far", FAR)
def test_values(dtype, v, far):
    x = _rows(v, dtype, far)
    ids = [v // 2, 0, v - 1, 1, v - 1, 2, v // 3, v // 3]
    top = min(v, 20)
    got = ojasx_amd.token_logprobs(x.to(DEV), torch.tensor(ids, device=DEV), top_k=top)
    lp, h, lse, best, order, _ = P.logprobs(x.double().numpy(), ids, top)
    sums = v / 64 + 64

    def near(a, b, tol):
        a = a.double().cpu().numpy()
        assert np.isfinite(a).all()
        assert (np.abs(a - b) <= tol).all(), float((np.abs(a - b) / tol).max())

    near(got.logprob, lp, ULP * (np.abs(lp) + sums))
    near(got.lse, lse, ULP * (np.abs(lse) + sums))
    near(got.entropy, h, ULP * sums * (1 + np.log(v)))
    near(got.top_logprobs, best, ULP * (np.abs(best) + sums))
    assert np.array_equal(got.top_ids.cpu().numpy(), order)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [6, 3001])
@pytest.mark.parametrize("far", FAR)
def test_gradient(dtype, v, far):
    _check_grad(_rows(v, dtype, far), [v // 2, 0, v - 1, 1, v - 1, 2, v // 3, v // 3], min(v, 5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("far", FAR)
def test_rows_without_alternatives_over_many_workgroups(dtype, far):
    x = _rows(128256, dtype, far)
    ids = [0] * 8
    got = ojasx_amd.token_logprobs(x.to(DEV), torch.tensor(ids, device=DEV))
    _, h, lse, _, _, _ = P.logprobs(x.double().numpy(), ids, 0)
    sums = 128256 / 64 + 64
    assert (np.abs(got.lse.double().cpu().numpy() - lse) <= ULP * (np.abs(lse) + sums)).all()
    assert (np.abs(got.entropy.double().cpu().numpy() - h) <= ULP * sums * 13).all()
