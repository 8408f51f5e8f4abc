"""The example decoder's rotations, before the cache and on the way into it, at positions near and far."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import rotary_plain as R
from test_gpu_cached_decoder import _example

pytestmark = pytest.mark.gpu


class Keeps:
    """A cache that keeps what it is given."""

    def append(self, k, v, slots):
        self.k, self.v = k, v

    def attention(self, q, *_, **__):
        self.q = q
        return torch.zeros_like(q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [0, 30000, 10 ** 6, 2 ** 31 - 40])
def test_rotated_queries_and_keys(dtype, first):
    model = _example().Decoder(layers=1, hidden=128, heads=6, kv_heads=2, head_dim=48, vocabulary=333, dtype=dtype)
    n = 37
    tokens = torch.arange(n, device="cuda") * 7 % 333
    pos = torch.arange(first, first + n, device="cuda").int()
    plan = SimpleNamespace(positions=pos, slots=None, seq_lens=None, query_starts=None)
    cache = Keeps()
    with torch.no_grad():
        model.hidden(tokens, plan, None, [cache])
        x = model.embedding[tokens]
        q, k, v = model.qkv[0](torch.nn.functional.rms_norm(x, x.shape[-1:])).split([288, 96, 96], -1)
    assert torch.equal(cache.v, v.unflatten(-1, (2, 48)))
    for got, raw in ((cache.q, q), (cache.k, k)):
        want, bound = R.rotate(raw.unflatten(-1, (-1, 48)).double().cpu().numpy(),
                               model.rotation.rates.cpu().numpy(), pos.cpu().numpy())
        err = np.abs(got.double().cpu().numpy() - want)
        assert got.dtype == dtype
        assert (err <= bound + torch.finfo(dtype).eps / 2 * (np.abs(want) + bound)).all()
