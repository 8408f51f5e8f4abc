"""What rounding weights to fewer bits may cost, where most of the weight lies on a key whose value is
zero and the output is made of the others' small weights.

Rows of q are 0 and +-1, which 16-bit fixed point holds exactly, so a score is off by its fp32
roundings only: (d + 4) * 2^-24 of the sum of |products|, and so is a weight, twice that.  With p_j
the softmax's weights, v_j the values, s_j a value's scale, and e_j = p_j s_j:
* few rows: 16-bit fixed point of the largest e_j of the key's 64: 127 / 65024 of that for each key;
* many rows: fp16 of e_j over a reference no larger than the largest: 2^-11 p_j |v_j| for each key, or
  where that is denormal 2^-25 * 127 of the largest e_j;
* fp32 rows: 2^-22 p_j |v_j|.
Sums of n terms in 32 bits add n * 2^-24 of the sum of |terms|, and the output is rounded to its type.
"""

import numpy as np
import pytest
import torch

import kv8_plain as P
from test_gpu_kv8 import DEV, DTYPES, HALF_ULP, _batch, _i32, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,group", [([1, 1], 4), ([3, 2], 4), ([60, 90], 2)])
@pytest.mark.parametrize("bits", [2, 8, 12, 14, 17, 20])
def test_small_weights_beside_a_large_one(dtype, new, group, bits):
    block, d, ctx = 64, 64, [700, 2500]
    tables, lens, starts, total = _batch(ctx, new, block)
    cache = _make(block, 1, d, total)
    k, v = P.codes_of(cache)
    rng = np.random.RandomState(bits)
    pattern = rng.choice([-1, 1], d)
    k[:] = rng.randint(-3, 4, k.shape)
    for r in range(len(ctx)):  # the third token of each request: a large key, a value of zero
        k[tables[r][0], 0, 2, :d] = 127 * pattern
        v[tables[r][0], 0, 2] = 0
    for codes, at in ((k, cache.k_codes), (v, cache.v_codes)):
        byte = P.byte_maps(block, d)[0 if codes is k else 1]
        flat = np.zeros((total, 1, block * d), np.int8)
        flat[:, :, byte.reshape(-1)] = codes.reshape(total, 1, -1)
        at.copy_(torch.from_numpy(flat).view(at.shape))
    cache.scales[:, :, 0] = 2.0 ** -7
    mask = rng.rand(starts[-1], group, d) < 0.5
    q = torch.from_numpy(np.where(mask, pattern, 0)).to(dtype).to(DEV)
    # the large key's score is about `bits` powers of two over the others
    scale = float(np.float32(bits * np.log(2) / (127 * 2.0 ** -7 * d / 2)))
    out = cache.attention(q, _i32(tables), _i32(lens), None if max(new) == 1 else _i32(starts),
                          scale=scale, max_query_len=max(new), max_seq_len=max(lens))
    out = out.double().cpu().numpy()
    vs = cache.scales.double().cpu().numpy()[:, 0, 1]
    many = max(new) * group > 48
    for r, table in enumerate(tables):
        for i in range(starts[r], starts[r + 1]):
            n = lens[r] - (starts[r + 1] - i) + 1
            j = np.arange(n)
            b = np.array(table)[j // block]
            kk, s = k[b, 0, j % block, :d] * 2.0 ** -7, vs[b]
            vv = v[b, 0, j % block, :d] * s[:, None]
            for h in range(group):
                x = kk @ np.where(mask[i, h], pattern, 0) * scale
                p = np.exp(x - x.max())
                p /= p.sum()
                want, size = p @ vv, p @ np.abs(vv)
                e = p * s
                score = (d + 4) * 2.0 ** -24 * scale * np.abs(kk).sum(1).max()
                bound = (4 * score + n * 2.0 ** -23 + 2.0 ** -20) * size
                if dtype == torch.float32:
                    bound = bound + 2.0 ** -22 * size
                elif many:
                    bound = bound + 2.0 ** -11 * size + n * 2.0 ** -25 * 127 * e.max()
                else:
                    tiles = [e[t:t + 64].max() for t in range(0, n, 64)]
                    bound = bound + 64 * 127 / 65024 * sum(tiles)
                bound = bound + HALF_ULP[dtype] * (np.abs(want) + bound) + 2.0 ** -25
                assert (np.abs(out[i, h] - want) <= bound).all()
