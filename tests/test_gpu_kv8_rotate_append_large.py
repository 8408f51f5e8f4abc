"""Rotated appends of many tokens, whose waves look for runs in windows of 16 or 32 tokens: to the bit what
rotating in fp32 and appending give, and the definition in 64 bits."""

import numpy as np
import pytest
import torch

import ojasx_amd
import rotary_plain as R
from ojasx_amd import rotary
from test_gpu_kv8 import DEV, _runs
from test_gpu_kv8_rotate_append import _check

pytestmark = pytest.mark.gpu


def _ragged(rng, tokens, block):
    """(slots, blocks): runs that begin and end anywhere, many of them in a window, single tokens, whole
    blocks, tokens that are not stored between them and inside."""
    spec, n = [], 0
    while n < tokens:
        length = (1, 1, rng.randint(2, 8), rng.randint(2, 8), rng.randint(1, block + 1),
                  rng.randint(block, 4 * block))[rng.randint(6)]
        spec.append((rng.randint(block), length))
        n += length
    spec.append((0, 3 * block))
    blocks = sum((off + length - 1) // block + 1 for off, length in spec)
    slots = []
    for s in _runs(rng, blocks, block, spec):
        if slots and s != slots[-1] + 1 and rng.rand() < 0.2:
            slots += [(-1, -7, blocks * block, 10 ** 12)[rng.randint(4)]] * rng.randint(1, 4)
        slots.append(s)
    for at in rng.randint(0, len(slots), 3):  # a run cut short: what follows of its block goes as well
        cut = slots[at] // block
        slots[at:] = [-1 if s // block == cut else s for s in slots[at:]]
    return slots, blocks


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("block,d,rot,heads,hq", [
    (16, 80, 40, 8, 16), (16, 128, 128, 5, 20), (16, 64, 64, 1, 4), (32, 64, 32, 2, 2),  # runs in registers
    (32, 64, 40, 3, 7),                                        # queries by 8 bytes or less beside them
    (64, 128, 128, 1, 4), (64, 128, 64, 2, 8), (64, 128, 128, 8, 16), (64, 256, 256, 2, 8),
    (128, 128, 64, 5, 10), (128, 192, 144, 2, 4), (256, 64, 64, 1, 2), (256, 128, 128, 2, 2),
    (256, 256, 128, 5, 5), (16, 256, 256, 2, 4), (16, 192, 64, 1, 3),
    (64, 72, 10, 2, 4), (16, 100, 100, 3, 3), (256, 33, 32, 4, 2), (64, 40, 24, 1, 1)])
def test_many_tokens(dtype, interleaved, block, d, rot, heads, hq):
    rng = np.random.RandomState(d + block + heads)
    g = torch.Generator().manual_seed(d + heads)
    slots, blocks = _ragged(rng, 16384 // (2 * heads) + 50, block)
    t = len(slots)
    assert t * 2 * heads > 16384
    r = rotary.rotation(rot, interleaved=interleaved, device=DEV)._replace(gain=1.1)
    # tokens from far under the blocks' scales to over them
    size = torch.exp2(torch.randint(-5, 4, (t, 1, 1), generator=g).float())
    x = (torch.randn(t, hq + 2 * heads, d, generator=g) * size).to(dtype).to(DEV)
    pos = torch.randint(0, 200000, (t,), generator=g, dtype=torch.int32).to(DEV)
    _check(x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:], pos, slots, r, blocks, block)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block,d,rot,heads,t", [(16, 64, 64, 8, 20000), (64, 64, 32, 9, 14000),
                                                 (256, 128, 64, 12, 11000)])
def test_more_windows_than_workgroups(dtype, block, d, rot, heads, t):
    assert -(-t // (16 if block < 64 else 32)) * -(-heads // 4) > 1024
    rng, g = np.random.RandomState(t), torch.Generator().manual_seed(t)
    slots, blocks = _ragged(rng, t, block)
    x = torch.randn(len(slots), 1 + 2 * heads, d, generator=g).to(dtype).to(DEV)
    pos = torch.randint(-5, 10 ** 6, (len(slots),), generator=g).to(DEV)
    _check(x[:, :1], x[:, 1:1 + heads], x[:, 1 + heads:], pos, slots, rotary.rotation(rot, device=DEV), blocks,
           block)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block,d,rot,heads,t", [(64, 128, 128, 8, 2100), (256, 64, 64, 1, 9001),
                                                 (128, 128, 64, 2, 4501), (16, 80, 40, 3, 2800)])
def test_many_tokens_by_the_definition(dtype, block, d, rot, heads, t):
    """Keys and values read back against those in 64 bits: half a step of the block's largest one, and what
    32-bit products and the scale's and the code's roundings add (the bound and its reason are those of
    the small calls' test)."""
    assert t * 2 * heads > 16384
    g = torch.Generator().manual_seed(t)
    cache = ojasx_amd.KV8Cache(-(-t // block) + 3, heads, d, block, DEV)
    r = rotary.rotation(rot, device=DEV)
    x = torch.randn(t, 2 + 2 * heads, d, generator=g).to(dtype).to(DEV)
    pos = torch.arange(t, device=DEV) + 12345
    cache.rotate_append(x[:, :2], x[:, 2:2 + heads], x[:, 2 + heads:], pos,
                        torch.arange(t, device=DEV) + 2 * block, r)
    n = -(-t // block)
    got = cache.read(torch.arange(2, 2 + n, dtype=torch.int32, device=DEV), torch.float32)
    keys, bound = R.rotate(x[:, 2:2 + heads].cpu().double().numpy(), r.rates.cpu().numpy(), pos.cpu().numpy())
    values = x[:, 2 + heads:].cpu().double().numpy()
    for i, (want, extra) in enumerate(((keys, bound), (values, 0))):
        scales = got[2][:, :, i].cpu().double().numpy()
        scale = np.repeat(scales, block, 0)[:t, :, None]
        have = got[i].reshape(-1, heads, d)[:t].cpu().double().numpy()
        assert (np.abs(have - want) <= scale * (0.5 + 127 * 2.0 ** -21) + extra).all()
        most = np.abs(want).max(2)
        top = np.stack([most[j:j + block].max(0) for j in range(0, t, block)])
        np.testing.assert_allclose(scales, top / 127, rtol=2.0 ** -20)
