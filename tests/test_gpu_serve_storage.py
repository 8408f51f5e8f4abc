"""What a kept result of a call keeps with it, where results lie side by side in an allocation: 64
KiB at most, or results of about its own size: the three of each token of a plan (or the three of
its requests), the values of each row (20 bytes and their padding), the alternatives (12)."""

import pytest
import torch

import ojasx_amd
from ojasx_amd import kv8

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
MOST = 64 * 1024


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _held(results, parts):
    """parts: the results by the allocations they may share."""
    for part in parts:
        own = sum((t.numel() * t.element_size() + 15) // 16 * 16 for t in part)
        for t in part:
            assert t.untyped_storage().nbytes() <= max(own, MOST)
    for i, a in enumerate(results):
        for b in results[i + 1:]:
            if a.numel() and b.numel():
                lo, hi = sorted((a, b), key=lambda t: t.data_ptr())
                assert lo.data_ptr() + lo.numel() * lo.element_size() <= hi.data_ptr()


@pytest.mark.parametrize("tokens", [1, 64, 3000, 5000, 100000])
def test_plan(tokens):
    new = [tokens // 2, tokens - tokens // 2]
    tables = torch.zeros(2, tokens // 16 + 1, dtype=torch.int32, device=DEV)
    p = kv8.plan(_i32([0, 0]), _i32(new), tables, torch.arange(20000, dtype=torch.int32, device=DEV),
                 _i32([20000]), 16, tokens)
    _held(list(p), (p[:3], p[3:]))
    assert p.positions.tolist() == list(range(new[0])) + list(range(new[1]))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("rows,top", [(1, 0), (8, 64), (100, 20), (3000, 5), (4096, 64)])
def test_token_logprobs(rows, top, grad):
    x = torch.randn(rows, 100, device=DEV).requires_grad_(grad)
    out = ojasx_amd.token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device=DEV), top)
    got = [t.detach() for t in out]
    stats = torch.empty(rows, 2)  # not returned, beside the rows' values
    _held(got, ([*got[:3], stats], got[3:]))
    want = torch.log_softmax(x.detach().double(), -1)[:, 0]
    assert (out.logprob.detach() - want).abs().max() < 1e-4
