"""Attention where scores are so large that 32-bit floats hold their whole numbers only, or not
even those.

A row's only element other than zero is a power of two times +-1 (held exactly by every form of
the kernels), so a key's score is that times one of its codes and a scale common to all keys.  Each
d has one key with the largest code and one with the smallest, apart from the others by a step of
1/127 of the largest score at least, 1000 / 127 > 7 here: far more than the scores' rounding of 2^-21
of it.  So all weights but the best key's are under e^-7 and as exact as in a row of small scores.
Bound: 2^-9 of a weight for its rounding to fewer bits (16-bit fixed point of the largest of 64:
64 / 65024; fp16: 2^-11), 4 * 2^-21 * |score| for the exponents of weights that are not zero
(they are under e^-60 from |score| = 8000 on: 0.016), and the output's own rounding.
"""

import numpy as np
import pytest
import torch

import kv8_plain as P
from test_gpu_kv8 import DEV, DTYPES, HALF_ULP, _batch, _i32, _make

pytestmark = pytest.mark.gpu


def _case(new, d, block, size, dtype, group):
    """Cache, tables, lengths, starts, rows and the softmax's scale for best scores of `size`."""
    ctx = [150, 40, 700][:len(new)]
    tables, lens, starts, total = _batch(ctx, new, block)
    cache = _make(block, 1, d, total)
    k, _ = P.codes_of(cache)
    dp = k.shape[3]
    rng = np.random.RandomState(d)
    km, _ = P.byte_maps(block, dp)
    k[:] = rng.randint(-126, 127, k.shape)
    k[..., d // 2:] = rng.randint(2, 127, k[..., d // 2:].shape)  # all of one sign
    for r, c in enumerate(ctx):
        for j in range(d):
            a, b = rng.choice(c, 2, replace=False)
            k[tables[r][a // block], 0, a % block, j] = 127
            k[tables[r][b // block], 0, b % block, j] = -127 if j < d // 2 else 1
    flat = np.zeros((total, 1, block * dp), np.int8)
    flat[:, :, km.reshape(-1)] = k.reshape(total, 1, -1)
    cache.k_codes.copy_(torch.from_numpy(flat).view(cache.k_codes.shape))
    ks = 0.0137
    cache.scales[:, :, 0] = ks
    q = torch.zeros(starts[-1], group, d)
    at = torch.from_numpy(rng.randint(0, d, q.shape[:2]))
    sign = torch.where(torch.from_numpy(rng.rand(*q.shape[:2]) < 0.5), 1.0, -1.0)
    q.scatter_(2, at[..., None], 4 * sign[..., None])
    return cache, tables, lens, starts, q.to(dtype).to(DEV), size / (4 * 127 * ks)


SIZES = [1e3, 8e3, 3e4, 1e5, 2e5, 1e6, 1e7, 1e8, 3e8, 1e9, 1e12, 1e20, 1e28]


def _check(new, d, block, size, dtype, group, **kw):
    cache, tables, lens, starts, q, scale = _case(new, d, block, size, dtype, group)
    k, v = P.codes_of(cache)
    s = cache.scales.cpu().numpy()
    # the scale as the kernels get it
    scale = float(np.float32(scale))
    want, lse, _, vmax = P.attention(q.float().cpu().numpy(), k, v, s[:, :, 0], s[:, :, 1],
                                     tables, lens, starts, scale, 0, block)
    one = all(b - a == 1 for a, b in zip(starts, starts[1:]))
    got, got_lse = cache.attention(q, _i32(tables), _i32(lens), None if one else _i32(starts),
                                   scale=scale, return_lse=True, **kw)
    got, got_lse = got.double().cpu().numpy(), got_lse.double().cpu().numpy()
    assert np.isfinite(got).all() and np.isfinite(got_lse).all()
    slack = (2.0 ** -9 + (4 * 2.0 ** -21 * size if size < 8000 else 0.0)) * vmax[..., None]
    bound = slack + HALF_ULP[q.dtype] * (np.abs(want) + slack)
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    assert (np.abs(got_lse - lse) <= 2.0 ** -20 * size + 2.0 ** -9).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_few_rows(dtype, size):
    _check([1, 1, 1], 64, 16, size, dtype, 4)
    _check([1, 1, 1], 96, 64, size, dtype, 16)
    _check([3, 1, 2], 200, 32, size, dtype, 3)
    _check([5, 2], 64, 64, size, dtype, 6, max_query_len=5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_many_rows(dtype, size):
    _check([70, 9, 33], 64, 16, size, dtype, 4)
    _check([100, 90, 1], 128, 64, size, dtype, 2, max_query_len=100)
    _check([64, 64], 256, 32, size, dtype, 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 40, 3]])
def test_scores_beyond_32_bits_leave_a_row_its_keys(dtype, new):
    # no score is a finite float: the row still sees its keys
    cache, tables, lens, starts, q, _ = _case(new, 64, 16, 1.0, dtype, 4)
    cache.scales[:, :, 0] = 1e4
    out, lse = cache.attention(q, _i32(tables), _i32(lens), _i32(starts), scale=1e37,
                               return_lse=True)
    assert torch.isfinite(out).all() and not torch.isneginf(lse).any() and not lse.isnan().any()
    assert (out.abs().amax(-1) > 0).all()
