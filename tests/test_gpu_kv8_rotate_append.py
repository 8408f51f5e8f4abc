"""Keys and queries rotated on the way into the cache: to the bit what rotating in fp32 and
appending give, and the definition in 64 bits."""

import numpy as np
import pytest
import torch

import kv8_plain as P
import ojasx_amd
import rotary_plain as R
from ojasx_amd import _native as N
from ojasx_amd import kv8, rotary, serve_ops as S
from test_gpu_kv8 import DEV, _runs

pytestmark = pytest.mark.gpu


def _caches(blocks, heads, d, block, seed, n=2):
    out = [ojasx_amd.KV8Cache(blocks, heads, d, block, DEV) for _ in range(n)]
    for c in out:
        P.fill(c, torch.Generator().manual_seed(seed))
    return out


def _check(q, k, v, pos, slots, r, blocks, block, seed=0):
    """One call against: queries by rotary.rotate, keys rotated in fp32 and appended in fp32,
    values appended as they are."""
    a, b = _caches(blocks, k.shape[1], k.shape[2], block, seed)
    slots = torch.as_tensor(slots, dtype=torch.int64, device=DEV)
    got = a.rotate_append(q, k, v, pos, slots, r)
    assert got.dtype == q.dtype and torch.equal(got, rotary.rotate(q, pos, r))
    other, = _caches(blocks, k.shape[1], k.shape[2], block, seed, 1)
    turned = rotary.rotate(k.float(), pos, r)
    other.append(turned, torch.zeros_like(turned), slots)
    b.append(k, v, slots)
    assert torch.equal(a.k_codes, other.k_codes)
    assert torch.equal(a.scales[..., 0], other.scales[..., 0])
    assert torch.equal(a.v_codes, b.v_codes)
    assert torch.equal(a.scales[..., 1], b.scales[..., 1])
    return a


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("block,d,rot,heads,hq", [
    (64, 128, 128, 2, 8), (16, 80, 40, 3, 3), (16, 80, 80, 1, 5), (32, 96, 32, 2, 2), (16, 64, 64, 5, 10),
    (256, 128, 64, 1, 4), (128, 256, 256, 1, 1), (256, 256, 64, 1, 2), (64, 72, 48, 2, 4), (64, 72, 8, 1, 1),
    (32, 33, 32, 2, 2), (16, 8, 8, 1, 3), (128, 192, 144, 1, 7), (16, 100, 100, 2, 2), (64, 16, 16, 2, 2),
    (32, 24, 16, 1, 2), (64, 1 + 1, 2, 1, 1)])
def test_runs_of_every_kind(dtype, interleaved, block, d, rot, heads, hq):
    rng = np.random.RandomState(d + block)
    g = torch.Generator().manual_seed(d)
    r = rotary.rotation(rot, interleaved=interleaved, device=DEV)._replace(gain=1.1)
    # a block, two more and a token, the rest of one, single tokens in the middle and at the end
    slots = _runs(rng, 16, block, [(0, block), (0, 2 * block + 1), (3, block - 3), (block // 2 + 1, 1),
                                   (block - 1, 1), (5, 2)])
    t = len(slots)
    x = (torch.randn(t, hq + 2 * heads, d, generator=g) * 2).to(dtype).to(DEV)
    x[-1] *= 3
    pos = torch.randint(0, 200000, (t,), generator=g, dtype=torch.int32).to(DEV)
    _check(x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:], pos, slots, r, 16, block)


@pytest.mark.parametrize("d,rot", [(80, 40), (128, 128), (48, 32)])
def test_the_definition(d, rot):
    """Keys read back against rotated ones in 64 bits: half a step of the block's largest key, and
    what 32-bit products and the scale's and the code's roundings add."""
    g = torch.Generator().manual_seed(3)
    block, t = 16, 75
    cache = ojasx_amd.KV8Cache(8, 2, d, block, DEV)
    r = rotary.rotation(rot, device=DEV)
    x = torch.randn(t, 6, d, generator=g).to(torch.bfloat16).to(DEV)
    pos = torch.arange(t, device=DEV) + 12345
    slots = torch.arange(t, device=DEV) + 2 * block
    cache.rotate_append(x[:, :2], x[:, 2:4], x[:, 4:], pos, slots, r)
    k, v, scales = cache.read(torch.arange(2, 7, dtype=torch.int32, device=DEV), torch.float32)
    want, bound = R.rotate(x[:, 2:4].cpu().double().numpy(), r.rates.cpu().numpy(), pos.cpu().numpy())
    scale = np.repeat(scales[:, :, 0].cpu().double().numpy(), block, 0)[:t, :, None]
    got = k.reshape(-1, 2, d)[:t].cpu().double().numpy()
    # at code 127 the product with the inverse scale may be off by 127 * 3 * 2^-24 of a step
    assert (np.abs(got - want) <= scale * (0.5 + 127 * 2.0 ** -21) + bound).all()
    most = np.abs(want).reshape(t, 2, d).max(2)
    top = np.stack([most[i:i + block].max(0) for i in range(0, t, block)])
    np.testing.assert_allclose(scales[:, :, 0].cpu().numpy(), top / 127, rtol=2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_elements_that_are_not_finite(dtype):
    g = torch.Generator().manual_seed(4)
    for d, rot, inter in ((64, 64, False), (64, 32, True), (40, 40, False)):
        x = torch.randn(20, 4, d, generator=g).to(dtype)
        x[3, 1, 5] = float("inf")
        x[7, 1, 0] = float("nan")
        x[9, 3, 2] = float("-inf")
        x[16:, 2] = 0
        x = x.to(DEV)
        r = rotary.rotation(rot, interleaved=inter, device=DEV)
        pos = torch.arange(20, device=DEV) * 7
        _check(x[:, 2:3].contiguous(), x[:, 1:3], x[:, 2:4], pos, list(range(16, 36)), r, 4, 16)
        x[:, 1] = 0  # a run of zeros beside one that raises a scale
        _check(x[:, :1], x[:, 1:2], x[:, 3:], pos, list(range(4, 24)), r, 4, 16)


def test_rows_that_are_views():
    g = torch.Generator().manual_seed(6)
    t, heads, d = 30, 3, 64
    base = torch.randn(2 * t, 5 * heads, d + 8, generator=g).to(torch.bfloat16).to(DEV)
    r = rotary.rotation(32, device=DEV)
    slots = [-1, 7] + list(range(64, 64 + t - 4)) + [200, 9000]
    for x in (base[:t, :, :d], base[::2, :, 3:d + 3], base[:t, ::2, 8:], base[:t, 1:, 1:d + 1]):
        pos = torch.arange(2 * t, device=DEV, dtype=torch.int32)[::2] * 3
        _check(x[:, :heads], x[:, heads:2 * heads], x[:, -heads:], pos, slots, r, 6, 64)
    apart = torch.randn(t, d, 6, generator=g).half().to(DEV).transpose(1, 2)
    _check(apart[:, :2], apart[:, 2:4], apart[:, 4:], pos.long(), slots, r, 6, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_heads_that_overlap(dtype):
    """Windows of one tensor as queries, keys and values."""
    t, d, r = 21, 16, rotary.rotation(16, device=DEV)
    flat = torch.randn(t, 18, device=DEV).to(dtype)
    x = flat.unfold(1, d, 1)
    assert x.shape == (t, 3, d) and x.stride()[1:] == (1, 1)
    pos, slots = torch.arange(t, device=DEV) * 77, torch.arange(t, device=DEV) + 5
    _check(x, x[:, :2], x[:, 1:], pos, slots, r, 4, 16)
    c, e = _caches(4, 2, d, 16, 0)
    a = c.rotate_append(x, x[:, :2], x[:, 1:], pos, slots, r)
    b = S.kv8_rotate_append(x, x[:, :2], x[:, 1:], pos, slots, r.rates, r.gain, False, e.k_codes,
                            e.v_codes, e.scales)
    assert a.stride(-1) == b.stride(-1) == 1 and torch.equal(a, b)
    dense = flat.unfold(1, d, 1).contiguous()
    assert torch.equal(a, rotary.rotate(dense, pos, r))


def test_no_tokens_and_padding():
    c, d = _caches(4, 2, 64, 16, 1)
    r = rotary.rotation(64, device=DEV)
    x = torch.zeros(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert c.rotate_append(x, x, x, none, none, r).shape == x.shape
    x = torch.randn(5, 2, 64, device=DEV, dtype=torch.bfloat16)
    skip = torch.full((5,), -1, device=DEV)
    q = c.rotate_append(x, x, x, skip, skip, r)   # padded tokens: position and slot -1
    assert torch.equal(q, rotary.rotate(x, skip, r))
    for a, b in ((c.k_codes, d.k_codes), (c.v_codes, d.v_codes), (c.scales, d.scales)):
        assert torch.equal(a, b)


def test_native_call_matches_the_op_and_refusals():
    r = rotary.rotation(64, device=DEV)
    x = torch.randn(20, 4, 96, device=DEV, dtype=torch.float16)
    pos, slots = torch.arange(20, device=DEV), torch.arange(20, device=DEV) + 3
    c, d = _caches(4, 1, 96, 16, 2)
    version = c.k_codes._version
    got = c.rotate_append(x[:, :2], x[:, 2:3], x[:, 3:], pos, slots, r)
    want = S.kv8_rotate_append(x[:, :2], x[:, 2:3], x[:, 3:], pos, slots, r.rates, 1.0, False, d.k_codes,
                               d.v_codes, d.scales)
    assert c.k_codes._version > version
    assert torch.equal(got, want) and got.stride() == want.stride()
    assert torch.equal(c.k_codes, d.k_codes) and torch.equal(c.scales, d.scales)
    good = (x[:, :2], x[:, 2:3], x[:, 3:], pos, slots, r)
    for i, bad in ((0, x[:19, :2]), (0, x[:, :2].float()), (0, x[:, :2, :64]), (0, x[:, 0]),
                   (1, x[:, :2]), (1, x[:, 2:3].bfloat16()), (3, pos[:19]), (3, pos.float()),
                   (3, pos[None]), (3, pos.cpu()), (4, slots.int()), (4, slots[:3]),
                   (5, rotary.rotation(98, device=DEV)), (5, rotary.rotation(64, device="cpu"))):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            c.rotate_append(*args)
    with pytest.raises(RuntimeError):  # no gradient passes the cache
        c.rotate_append(x[:, :2].clone().requires_grad_(True), *good[1:]).float().sum().backward()


def test_no_queries_and_compiled_calls():
    r = rotary.rotation(64, device=DEV)
    x = torch.randn(20, 4, 96, device=DEV, dtype=torch.bfloat16)
    pos, slots = torch.arange(20, device=DEV), torch.arange(20, device=DEV) + 3
    c, d, e = _caches(4, 1, 96, 16, 2, 3)
    want = c.rotate_append(x[:, :2], x[:, 2:3], x[:, 3:], pos, slots, r)
    none = d.rotate_append(x[:, :0], x[:, 2:3], x[:, 3:], pos, slots, r)
    assert none.shape == (20, 0, 96) and torch.equal(c.k_codes, d.k_codes)
    f = torch.compile(lambda q: kv8.rotate_append(q, x[:, 2:3], x[:, 3:], pos, slots, r, e.k_codes,
                                                  e.v_codes, e.scales) * 1, backend="eager")
    assert torch.equal(f(x[:, :2]), want) and torch.equal(c.k_codes, e.k_codes)
    g = torch.compile(lambda p: kv8.reorder(p, pos[:2].int() + 20, slots[:4].int().view(2, 2),
                                            slots[:3].int(), slots[:1].int(), 16, 9).block_tables * 1,
                      backend="eager")
    rows = torch.tensor([1, 1, 0], device=DEV)
    assert torch.equal(g(rows), kv8.reorder(rows, pos[:2].int() + 20, slots[:4].int().view(2, 2),
                                            slots[:3].int(), slots[:1].int(), 16, 9).block_tables)


def test_in_a_graph_and_on_a_stream():
    r = rotary.rotation(128, device=DEV)
    x = torch.randn(9, 6, 128, device=DEV, dtype=torch.bfloat16)
    pos, slots = torch.arange(9, device=DEV), torch.arange(9, device=DEV)
    c, d = _caches(8, 1, 128, 64, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.rotate_append(x[:, :4], x[:, 4:5], x[:, 5:], pos, slots, r)
    torch.cuda.current_stream().wait_stream(side)
    d.rotate_append(x[:, :4], x[:, 4:5], x[:, 5:], pos, slots, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.rotate_append(x[:, :4], x[:, 4:5], x[:, 5:], pos, slots, r)
    for i in range(4):
        x.copy_(torch.randn(9, 6, 128, device=DEV))
        pos += 9
        slots += 9
        graph.replay()
        torch.cuda.synchronize()
        want = d.rotate_append(x[:, :4], x[:, 4:5], x[:, 5:], pos, slots, r)
        assert torch.equal(out, want)
        for a, b in ((c.k_codes, d.k_codes), (c.v_codes, d.v_codes), (c.scales, d.scales)):
            assert torch.equal(a, b)
