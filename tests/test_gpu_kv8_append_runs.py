"""Whole blocks and long runs appended at every head size on the 16-byte grid."""

import numpy as np
import pytest
import torch

import kv8_plain as P
import ojasx_amd
from test_gpu_kv8 import DEV, _check_append, _runs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
def test_every_head_size_on_the_grid(dtype, block):
    rng = np.random.RandomState(block)
    for d in range(8, 257, 8):
        g = torch.Generator().manual_seed(d + block)
        cache = ojasx_amd.KV8Cache(8, 2, d, block, DEV)
        P.fill(cache, g)
        # a block, two more and a token, the rest of one, its second half
        slots = _runs(rng, 8, block, [(0, block), (0, 2 * block + 1), (3, block - 3),
                                      (block // 2 + 1, block // 2 - 1)])
        k, v = (torch.randn(2, len(slots), 2, d, generator=g) * 2).to(dtype).to(DEV).unbind(0)
        # the largest key of a run at its end
        k[-1] *= 3
        _check_append(cache, k, v, slots)
