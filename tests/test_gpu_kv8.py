"""The 8-bit paged cache and its attention on the GPU against the plain forms of kv8_plain.

Bounds of attention, derived from the kernel's number formats (no result of it went into them):
q is rounded to 16-bit fixed point of its row's largest value a, an error of a / 65024 an element
at most, so a score is off by e = |scale| * a * max_j sum_d |k_jd| / 65024 and a weight by the
factor exp(2 e); weights are rounded to 16-bit fixed point of the largest in their 64 keys, 64 *
(1 / 65024) of it at most in sum, and multiply values of at most 127 scales.  fp32 sums of n
terms add n * 2^-24, and the output is rounded to its type.  fp32 rows are computed in fp32 or
finer throughout: the scores' error is d + 4 roundings of the largest sum of |products|.
"""

import math

import numpy as np
import pytest
import torch

import kv8_plain as P
import ojasx_amd
from ojasx_amd import kv8

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ plan

def _plan_both(seq, new, width, free, num_free, block, tokens):
    r = len(seq)
    tables = [[1000 * i + j if j < -(-max(s, 0) // block) else -1 for j in range(width)]
              for i, s in enumerate(seq)]
    got_tables = torch.tensor(tables, dtype=torch.int32, device=DEV).reshape(r, width)
    p = kv8.plan(_i32(seq).reshape(r), _i32(new).reshape(r), got_tables, _i32(free).reshape(-1),
                 _i32([num_free]), block, tokens)
    want = P.plan(seq, new, tables, free, num_free, block, tokens)
    got = (got_tables.tolist(), p.slots.tolist(), p.positions.tolist(), p.requests.tolist(),
           p.query_starts.tolist(), p.seq_lens.tolist(), p.num_free.item())
    names = ("tables", "slots", "positions", "requests", "starts", "lens", "num_free")
    for name, g, w in zip(names, got, want):
        assert g == w, name


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("r,hi", [(1, 1), (3, 40), (65, 1), (200, 300), (4096, 3), (4097, 2),
                                  (9001, 2)])
def test_plan(block, r, hi):
    rng = np.random.RandomState(r + hi)
    seq = rng.randint(0, 3 * block, r).tolist()
    new = rng.randint(0, hi + 1, r).tolist()
    total = sum(new)
    width = max(-(-(s + n) // block) for s, n in zip(seq, new)) + 1
    free = rng.permutation(100000)[:total + r].tolist()
    _plan_both(seq, new, width, free, len(free), block, total)


def test_plan_edges():
    # no request; no token; whole blocks; padding; too few tokens; negative lengths
    _plan_both([], [], 0, [], 0, 16, 0)
    _plan_both([], [], 4, [5], 1, 16, 7)
    _plan_both([0, 5], [0, 0], 2, [9, 8], 2, 16, 0)
    _plan_both([16, 32, 0, 15], [16, 1, 16, 1], 4, list(range(50, 60)), 10, 16, 34)
    _plan_both([3, 4], [5, 6], 2, [1, 2], 2, 16, 20)
    _plan_both([3, 4, 9], [5, 20, 6], 3, [1, 2, 3, 4], 4, 16, 12)
    _plan_both([-3, 4], [5, -6], 2, [1, 2], 2, 16, 5)
    # the stack runs out, is empty, claims more than it holds; a table too narrow
    _plan_both([0, 0, 16], [40, 40, 40], 4, [7, 6, 5], 3, 16, 120)
    _plan_both([10], [40], 4, [], 0, 16, 40)
    _plan_both([10], [40], 4, [3, 4], 9, 16, 40)
    _plan_both([10, 20], [60, 5], 2, [3, 4, 5], 3, 16, 65)
    _plan_both([40, 20], [60, 5], 2, [3, 4, 5], 3, 16, 65)


def test_plan_of_a_strided_table_and_a_chain_of_steps():
    wide = torch.full((3, 10), -7, dtype=torch.int32, device=DEV)
    tables = wide[:, 2:8]
    lens, left = _i32([0, 0, 0]), _i32([20])
    free = _i32(list(range(20)))
    seen = []
    for new in ([30, 1, 0], [1, 1, 1], [17, 0, 40]):
        p = kv8.plan(lens, _i32(new), tables, free, left, 16, sum(new))
        seen += p.slots.tolist()
        lens, left = p.seq_lens, p.num_free
    assert len(set(seen)) == len(seen) == 91 and min(seen) >= 0
    assert lens.tolist() == [48, 2, 41] and left.item() == 20 - 3 - 1 - 3
    assert (wide[:, :2] == -7).all() and (wide[:, 8:] == -7).all()


# ------------------------------------------------------------------ append, read

def _runs(rng, total_blocks, block, spec):
    """Slots of runs (offset, length) in random blocks."""
    free = iter(rng.permutation(total_blocks).tolist())
    slots = []
    for off, n in spec:
        b = next(free)
        while n > 0:
            k = min(n, block - off)
            slots += [b * block + off + i for i in range(k)]
            n, off = n - k, 0
            b = next(free) if n else b
    return slots


def _check_append(cache, k, v, slots):
    want_k, want_v = P.codes_of(cache)
    sc = cache.scales.cpu().numpy().copy()
    cache.append(k, v, torch.tensor(slots, dtype=torch.int64, device=DEV))
    for i, (codes, x) in enumerate(((want_k, k), (want_v, v))):
        s = sc[:, :, i].copy()
        P.append(codes, s, x.float().cpu().numpy(), slots, cache.block_size)
        sc[:, :, i] = s
    got_k, got_v = P.codes_of(cache)
    d = cache.head_dim
    assert np.array_equal(cache.scales.cpu().numpy(), sc)
    assert np.array_equal(got_k[..., :d], want_k[..., :d])
    assert np.array_equal(got_v[..., :d], want_v[..., :d])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,heads,d", [(16, 1, 64), (16, 3, 80), (32, 2, 128), (64, 2, 1),
                                           (64, 1, 33), (128, 2, 96), (256, 1, 256), (64, 3, 200)])
def test_append(dtype, block, heads, d):
    rng = np.random.RandomState(d + block)
    g = torch.Generator().manual_seed(d)
    cache = ojasx_amd.KV8Cache(40, heads, d, block, DEV)
    P.fill(cache, g)
    spec = [(0, 1), (5, 1), (block - 1, 1), (0, block), (3, block - 3), (7, 2), (15, 1),
            (9, block + 4), (0, 2 * block + 1)]
    slots = _runs(rng, 40, block, spec)
    # elements from far under the blocks' scales to over them
    size = torch.exp2(torch.randint(-6, 4, (len(slots), heads, 1), generator=g).float())
    k = (torch.randn(len(slots), heads, d, generator=g) * size).to(dtype).to(DEV)
    v = (torch.randn(len(slots), heads, d, generator=g) * size.flip(0)).to(dtype).to(DEV)
    _check_append(cache, k, v, slots)


def test_append_many_tokens_takes_wide_windows():
    rng = np.random.RandomState(3)
    heads, d, block = 8, 64, 16
    cache = ojasx_amd.KV8Cache(200, heads, d, block, DEV)
    slots = _runs(rng, 200, block, [(3, 700), (0, 500), (15, 2)] + [(i % 16, 1) for i in range(60)])
    assert len(slots) * 2 * heads > 16384
    k = torch.randn(len(slots), heads, d, device=DEV, dtype=torch.bfloat16)
    _check_append(cache, k, k * 2, slots)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_special_elements_and_skipped_slots(dtype):
    g = torch.Generator().manual_seed(1)
    cache = ojasx_amd.KV8Cache(6, 2, 64, 16, DEV)
    P.fill(cache, g)
    cache.scales[2] = 0
    n = 24
    x = torch.randn(n, 2, 64, generator=g)
    x[0, 0, 3], x[0, 0, 5], x[1, 1, 7] = math.inf, math.nan, -math.inf
    x[2] = 0                      # zeros into a fresh block
    x[3] = math.nan               # nothing finite
    x[4] = 2.0 ** -110            # too small for a scale
    x[5, 0] = math.inf
    slots = [0, 1, 16, 2 * 16 + 4, 3 * 16, 4 * 16, -1, 6 * 16, 6 * 16 + 1, -5, 10 ** 12] + \
        [5 * 16 + i for i in range(13)]
    k = x.to(dtype).to(DEV)
    _check_append(cache, k, k.flip(2).contiguous(), slots)


def test_append_of_strided_rows_and_on_another_stream():
    rng = np.random.RandomState(5)
    for pad in (0, 1):  # aligned rows of a fused projection; rows that start anywhere
        cache = ojasx_amd.KV8Cache(20, 2, 96, 16, DEV)
        slots = _runs(rng, 20, 16, [(2, 30), (0, 9), (4, 1)])
        qkv = torch.randn(len(slots), 2 * 96 * 3 + pad, device=DEV, dtype=torch.bfloat16)
        k = qkv[:, pad:][:, 192:384].unflatten(1, (2, 96))
        v = qkv[:, pad:][:, 384:576].unflatten(1, (2, 96))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _check_append(cache, k, v, slots)
        # heads apart further than tokens: [heads, tokens, d] storage
        kt = torch.randn(2, len(slots), 96, device=DEV, dtype=torch.bfloat16).transpose(0, 1)
        _check_append(cache, kt, kt, slots)
        # one head's element broadcast to both
        kb = torch.randn(len(slots), 1, 96, device=DEV, dtype=torch.bfloat16).expand(-1, 2, -1)
        _check_append(cache, kb, kb, slots)
        torch.cuda.current_stream().wait_stream(side)


def test_appending_one_by_one_keeps_values_within_their_roundings():
    # every growth of a scale rounds earlier codes again: half a step of each scale at most
    d, block = 64, 16
    cache = ojasx_amd.KV8Cache(1, 1, d, block, DEV)
    x = torch.randn(block, 1, d, device=DEV) * torch.linspace(0.2, 3, block, device=DEV)[:, None, None]
    scales = []
    for t in range(block):
        cache.append(x[t:t + 1], x[t:t + 1], torch.tensor([t], device=DEV))
        scales.append(cache.scales[0, 0, 0].item())
    k, v, s = cache.read(_i32([0]), torch.float32)
    assert torch.equal(k, v) and s[0, 0, 0].item() == scales[-1]
    for t in range(block):
        grown = sorted(set(scales[t:]))
        err = (k[0, t, 0] - x[t, 0]).abs().max().item()
        assert err <= 0.5 * sum(grown) * (1 + 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,heads,d", [(16, 1, 64), (32, 3, 80), (64, 2, 128), (128, 1, 33),
                                           (256, 2, 256), (16, 5, 1)])
def test_read(dtype, block, heads, d):
    g = torch.Generator().manual_seed(block + d)
    cache = ojasx_amd.KV8Cache(7, heads, d, block, DEV)
    P.fill(cache, g)
    blocks = [3, 6, 0, -1, 3, 7]
    k, v, s = cache.read(_i32(blocks), dtype)
    codes = P.codes_of(cache)
    sc = cache.scales.cpu().numpy()
    for i, (got, c) in enumerate(((k, codes[0]), (v, codes[1]))):
        assert got.shape == (6, block, heads, d) and got.dtype == dtype
        for n, b in enumerate(blocks):
            if not 0 <= b < 7:
                assert not got[n].any() and not s[n].any()
                continue
            want = torch.from_numpy(c[b, :, :, :d].astype(np.float32) * sc[b, :, i][:, None, None])
            assert torch.equal(got[n].cpu(), want.transpose(0, 1).to(dtype))
            assert torch.equal(s[n].cpu(), cache.scales[b].cpu())
    none = cache.read(_i32([]).reshape(0), dtype)
    assert none[0].shape == (0, block, heads, d)


# ------------------------------------------------------------------ attention

def _batch(ctx, new, block, extra=0):
    """Block tables over a shuffled pool, lengths, starts and the pool's size."""
    need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
    total = sum(need) + 3
    perm = np.random.RandomState(total).permutation(total).tolist()
    width = max(need + [1]) + extra
    tables, at = [], 0
    for n in need:
        tables.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return tables, [c + n for c, n in zip(ctx, new)], starts, total


def _check_attention(cache, q, tables, lens, starts, window=0, scale=None, call=None, **kw):
    d = q.shape[-1]
    sc = scale if scale is not None else d ** -0.5
    k, v = P.codes_of(cache)
    s = cache.scales.cpu().numpy()
    want, lse, reach, vmax = P.attention(q.float().cpu().numpy(), k, v, s[:, :, 0], s[:, :, 1],
                                         tables, lens, starts, sc, window, cache.block_size)
    one = all(b - a == 1 for a, b in zip(starts, starts[1:])) and kw.pop("decode", True)
    got, got_lse = (call or cache.attention)(
        q, _i32(tables), _i32(lens), None if one else _i32(starts), scale=scale, window=window,
        return_lse=True, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    got, got_lse = got.double().cpu().numpy(), got_lse.double().cpu().numpy()
    a = q.float().abs().amax(-1).double().cpu().numpy()
    n = max(lens + [1])
    if q.dtype == torch.float32:
        e = (d + 4) * 2.0 ** -24 * abs(sc) * a * reach + 2.0 ** -22
        fixed = 0.0
    else:
        e = abs(sc) * a * reach / 65024 + (d + 4) * 2.0 ** -24 * abs(sc) * a * reach + 2.0 ** -22
        fixed = 64 / 65024
    slack = (2 * e + fixed + n * 2.0 ** -23)[..., None] * vmax[..., None]
    bound = slack + HALF_ULP[q.dtype] * (np.abs(want) + slack) + 2.0 ** -25
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    seen = np.isfinite(lse)
    assert np.array_equal(np.isneginf(got_lse), ~seen)
    lse_bound = e + fixed + n * 2.0 ** -23 + 2.0 ** -22 * (1 + np.abs(np.where(seen, lse, 0)))
    assert (np.abs(got_lse[seen] - lse[seen]) <= lse_bound[seen]).all()


def _make(block, hkv, d, total, seed=0):
    cache = ojasx_amd.KV8Cache(total, hkv, d, block, DEV)
    P.fill(cache, torch.Generator().manual_seed(seed + d))
    return cache


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block,hkv,group,d", [
    (16, 1, 1, 64), (16, 2, 4, 128), (32, 2, 3, 80), (64, 1, 8, 128), (64, 2, 5, 192),
    (128, 1, 16, 256), (256, 1, 20, 64), (64, 1, 33, 128), (16, 3, 1, 1), (64, 1, 2, 17),
    (32, 1, 64, 96), (16, 1, 7, 200)])
def test_single_tokens(dtype, block, hkv, group, d):
    ctx = [0, 1, 14, 15, 16, 62, 63, 64, 65, 130, 300]
    new = [1] * len(ctx)
    tables, lens, starts, total = _batch(ctx, new, block, extra=1)
    cache = _make(block, hkv, d, total)
    q = (torch.randn(len(ctx), hkv * group, d) * 1.5).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block,hkv,group,d,new", [
    (16, 1, 1, 64, [1, 2, 3]), (64, 2, 4, 128, [5, 17, 64]), (32, 1, 3, 80, [33, 1, 90]),
    (64, 1, 8, 128, [40, 7]), (128, 1, 2, 256, [130, 20]), (16, 2, 1, 192, [65, 128, 0]),
    (64, 1, 16, 64, [3, 50]), (16, 1, 5, 33, [100])])
def test_several_tokens(dtype, block, hkv, group, d, new):
    ctx = [0, 37, 200][:len(new)]
    tables, lens, starts, total = _batch(ctx, new, block)
    cache = _make(block, hkv, d, total)
    q = torch.randn(starts[-1], hkv * group, d).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts)
    _check_attention(cache, q, tables, lens, starts, max_query_len=max(new), max_seq_len=max(lens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,group,d,new", [
    (2, 4, 128, [9, 1, 11, 4]), (1, 1, 64, [17, 33, 48, 2]), (1, 3, 200, [16, 7, 1, 12]),
    (1, 20, 80, [2, 1, 2, 0]), (2, 7, 96, [6, 5, 3, 1])])
def test_a_few_rows_of_a_request(dtype, hkv, group, d, new):
    # up to 48 of a key head: several tiles of a request in one launch, over few and many keys
    for ctx in ([0, 3, 60, 200], [700, 0, 64, 1500]):
        tables, lens, starts, total = _batch(ctx, new, 32)
        cache = _make(32, hkv, d, total)
        q = torch.randn(starts[-1], hkv * group, d).to(dtype).to(DEV)
        _check_attention(cache, q, tables, lens, starts, max_query_len=max(new))
        _check_attention(cache, q, tables, lens, starts, max_query_len=max(new), window=77)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv,group,d,new", [
    (2, 4, 128, [130, 3, 64]), (1, 2, 64, [200, 90, 1]), (2, 5, 40, [70, 26, 51]),
    (1, 4, 192, [90, 33, 2]), (1, 3, 256, [100, 44, 0]), (2, 1, 96, [256, 128, 129])])
def test_rows_under_long_bounds(dtype, hkv, group, d, new):
    # tables of many more columns than the requests use: the launch is sized for long ones
    tables, lens, starts, total = _batch([0, 300, 70], new, 64, extra=1100)
    cache = _make(64, hkv, d, total)
    q = torch.randn(starts[-1], hkv * group, d).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts)
    _check_attention(cache, q, tables, lens, starts, window=100, max_query_len=max(new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("extra", [0, 500])
def test_more_tiles_than_workgroups_at_a_time(dtype, extra):
    # also requests of equal length, which need no place for shorter ones
    ctx = [(37 * i) % 150 for i in range(90)]
    for new in ([(7 * i) % 23 + 1 for i in range(90)], [20] * 90):
        tables, lens, starts, total = _batch(ctx, new, 16, extra=extra)
        cache = _make(16, 6, 32, total)
        q = torch.randn(starts[-1], 18, 32).to(dtype).to(DEV)
        _check_attention(cache, q, tables, lens, starts, max_query_len=max(new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 65, 100, 1000])
def test_windows(dtype, window):
    ctx, new = [0, 5, 100, 333], [3, 1, 70, 2]
    tables, lens, starts, total = _batch(ctx, new, 32)
    cache = _make(32, 1, 64, total)
    q = torch.randn(starts[-1], 2, 64).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts, window=window)
    tables, lens, starts, total = _batch(ctx, [1] * 4, 32)
    _check_attention(cache, q[:4], tables, lens, starts, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts_are_split_and_joined(dtype):
    ctx = [5000, 9, 2047, 0, 700]
    tables, lens, starts, total = _batch(ctx, [1] * 5, 64, extra=40)
    cache = _make(64, 1, 128, total)
    q = torch.randn(5, 4, 128).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts)
    _check_attention(cache, q, tables, lens, starts, max_seq_len=max(lens))
    tables, lens, starts, total = _batch([4000, 30], [20, 3], 64)
    q = torch.randn(23, 4, 128).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts, max_query_len=20, max_seq_len=max(lens))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing(dtype):
    # lengths of zero, queries before the first key, blocks that are none (whole tiles of them too)
    cache = _make(16, 1, 64, 40)
    tables = [[-1] * 12, list(range(12)), [-1, -1, -1, -1, 5, 6] + [-1] * 6,
              [3, 40, 999, 2, 7, -2147483648] + [-1] * 6]
    q = torch.randn(4 + 3, 2, 64).to(dtype).to(DEV)
    _check_attention(cache, q, tables, [0, 2, 90, 85], [0, 1, 5, 6, 7])
    _check_attention(cache, q[:4], tables, [0, 2, 90, 85], [0, 1, 2, 3, 4])
    _check_attention(cache, q[:4], tables, [0, -3, 60, 85], [0, 1, 2, 3, 4])
    _check_attention(cache, q[:4], [t[:2] for t in tables], [5, 30, 90, 200], [0, 1, 2, 3, 4])
    out = cache.attention(q[:0], _i32(tables)[:0], _i32([]).reshape(0))
    assert out.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 0, 1], [1, 3, 2], [70, 5, 90]])
@pytest.mark.parametrize("d", [64, 100, 256])
def test_tokens_of_no_request_are_zero(dtype, new, d):
    tables, lens, starts, total = _batch([30, 0, 9], new, 16)
    cache = _make(16, 2, d, total)
    end = starts[-1]
    q = torch.randn(end + 300, 6, d).to(dtype).to(DEV)

    def call(_, tables, lens, starts, **kw):
        torch.full((4 * q.numel(),), math.nan, device=DEV)  # outputs take memory that held NaN
        out, lse = cache.attention(q, tables, lens, starts, **kw)
        assert not out[end:].any() and torch.isneginf(lse[end:]).all()
        return out[:end], lse[:end]

    _check_attention(cache, q[:end], tables, lens, starts, call=call)
    _check_attention(cache, q[:end], tables, lens, starts, call=call, max_query_len=max(new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales_of_the_softmax(dtype, scale):
    tables, lens, starts, total = _batch([100, 20], [1, 9], 16)
    cache = _make(16, 1, 64, total)
    q = torch.randn(10, 2, 64).to(dtype).to(DEV)
    _check_attention(cache, q, tables, lens, starts, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_queries_and_scales_of_blocks(dtype):
    tables, lens, starts, total = _batch([100, 20, 70], [1, 1, 1], 16)
    cache = _make(16, 1, 64, total)
    # blocks of zeros, far apart scales
    cache.scales[::3] *= 1e-12
    cache.scales[::4] = 0
    cache.scales[1::4] *= 30
    q = torch.randn(3, 2, 64)
    q[0] *= 1e-6
    q[1, 0] = 0
    q[2, 1, 5] = 50
    _check_attention(cache, q.to(dtype).to(DEV), tables, lens, starts)
    # NaN and infinities stay in their rows
    q = torch.randn(3, 2, 64)
    q[0, 0, 3], q[1, 1, 4], q[2, 0, 0] = math.nan, math.inf, -math.inf
    out, lse = cache.attention(q.to(dtype).to(DEV), _i32(tables), _i32(lens), return_lse=True)
    bad = torch.tensor([[True, False], [False, True], [True, False]])
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad)
    assert torch.equal(lse.isnan().cpu(), bad)


@pytest.mark.parametrize("new", [[1, 1, 1], [2, 5, 40]])
def test_strided_queries_tables_and_another_stream(new):
    tables, lens, starts, total = _batch([30, 100, 3], new, 16)
    cache = _make(16, 2, 80, total)
    for pad in (0, 1):
        qkv = torch.randn(starts[-1], 8 * 80 + pad, device=DEV, dtype=torch.bfloat16)
        q = qkv[:, pad:][:, :4 * 80].unflatten(1, (4, 80))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _check_attention(cache, q, tables, lens, starts)
        torch.cuda.current_stream().wait_stream(side)
    q = torch.randn(4, starts[-1], 80, device=DEV, dtype=torch.float16).transpose(0, 1)
    _check_attention(cache, q, tables, lens, starts)
    q = torch.randn(starts[-1], 80, 4, device=DEV, dtype=torch.float16).transpose(1, 2)
    _check_attention(cache, q, tables, lens, starts)

    def call(q, tables, lens, starts, **kw):
        wide = torch.full((3, 2 * tables.shape[1] + 5), 7, dtype=torch.int32, device=DEV)
        wide[:, 5:5 + tables.shape[1]] = tables
        out = cache.attention(q, wide[:, 5:5 + tables.shape[1]], lens, starts, **kw)
        every = torch.stack([tables, tables], 2).flatten(1)[:, ::2]
        again = cache.attention(q, every, lens, starts, **kw)
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
        return out

    _check_attention(cache, q, tables, lens, starts, call=call)


def test_results_repeat_bit_for_bit():
    tables, lens, starts, total = _batch([3000, 1500, 10], [1, 1, 1], 64)
    cache = _make(64, 2, 128, total)
    q = torch.randn(3, 8, 128, device=DEV, dtype=torch.bfloat16)
    first = cache.attention(q, _i32(tables), _i32(lens))
    for _ in range(5):
        assert torch.equal(first, cache.attention(q, _i32(tables), _i32(lens)))


def test_a_captured_step_replays():
    block, hkv, d = 16, 2, 64
    cache = ojasx_amd.KV8Cache(64, hkv, d, block, DEV)
    tables = torch.full((3, 20), -1, dtype=torch.int32, device=DEV)
    free, left, lens = _i32(list(range(64))), _i32([64]), _i32([0, 0, 0])
    ones = _i32([1, 1, 1])
    q = torch.zeros(3, 4, d, device=DEV, dtype=torch.bfloat16)
    k, v = torch.zeros(2, 3, hkv, d, device=DEV, dtype=torch.bfloat16).unbind(0)

    def step(cache, tables, lens, left):
        p = kv8.plan(lens, ones, tables, free, left, block, 3)
        cache.append(k, v, p.slots)
        o = cache.attention(q, tables, p.seq_lens)
        lens.copy_(p.seq_lens)
        left.copy_(p.num_free)
        return o

    other = ojasx_amd.KV8Cache(64, hkv, d, block, DEV)
    eager = (other, tables.clone(), lens.clone(), left.clone())
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(cache, tables, lens, left)
    torch.cuda.current_stream().wait_stream(warm)
    for t in (cache.k_codes, cache.v_codes, cache.scales, lens):
        t.zero_()
    tables.fill_(-1)
    left.fill_(64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(cache, tables, lens, left)
    for i in range(40):
        g = torch.Generator().manual_seed(i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, step(*eager)), i
    assert torch.equal(tables, eager[1]) and torch.equal(cache.k_codes, other.k_codes)


def test_offsets_past_32_bits():
    # 2.6 GB of codes: the last blocks' bytes lie beyond 2^31
    block, hkv, d = 64, 8, 128
    total = 40000
    cache = ojasx_amd.KV8Cache(total, hkv, d, block, DEV)
    assert cache.k_codes.numel() > 2 ** 31
    used = [total - 1, 3, total - 7]
    small = ojasx_amd.KV8Cache(3, hkv, d, block, DEV)
    k = torch.randn(150, hkv, d, device=DEV, dtype=torch.bfloat16)
    at = torch.arange(150, device=DEV)
    cache.append(k, -k, _i32(used).long()[at // block] * block + at % block)
    small.append(k, -k, at)
    q = torch.randn(2, 16, d, device=DEV, dtype=torch.bfloat16)
    for starts in (None, _i32([0, 2])):
        lens = _i32([150, 77]) if starts is None else _i32([150])
        n = lens.numel()
        a = cache.attention(q, _i32([used] * n), lens, starts)
        b = small.attention(q, _i32([[0, 1, 2]] * n), lens, starts)
        assert torch.equal(a, b)
    for a, b in zip(cache.read(_i32(used)), small.read(_i32([0, 1, 2]))):
        assert torch.equal(a[:2], b[:2])
