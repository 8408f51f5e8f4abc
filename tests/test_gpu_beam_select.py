"""Beam search's selection against the definition in 64 bits."""

import math

import numpy as np
import pytest
import torch

import beam_plain as P
import ojasx_amd
from ojasx_amd import _native as N
from ojasx_amd import beam_select, serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(x, scores, num, finished=None, pad=0):
    got = beam_select(x, scores, num, finished=finished, pad_id=pad)
    want = P.select(x.detach().float().cpu().numpy(), scores.cpu().numpy(), num,
                    None if finished is None else finished.cpu().numpy(), pad)
    assert np.array_equal(got.parents.cpu().numpy(), want[1])
    assert np.array_equal(got.tokens.cpu().numpy(), want[2])
    a, b = got.scores.cpu().numpy().astype(np.float64), want[0]
    assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isneginf(a), np.isneginf(b))
    on = np.isfinite(b)
    a, b = a[on], b[on]
    # one rounding, and what a sum that is partly 32-bit is off by where no near value asks for more
    assert (np.abs(a - b) <= 2.0 ** -24 * np.abs(b) + 2.0 ** -20).all()
    return got


def _logits(shape, g, width=2.0):
    x = torch.randn(shape, generator=g) * width
    return x + 8 * (torch.rand(shape, generator=g) > 0.998)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("g,k,v,num", [
    (1, 1, 1, 1), (1, 4, 3, 8), (2, 3, 5, 15), (3, 1, 1000, 1), (1, 4, 32000, 8), (5, 2, 8193, 4),
    (2, 5, 50021, 10), (1, 1, 128256, 64), (1, 64, 2050, 64), (2, 17, 777, 34), (70, 8, 1025, 16),
    (300, 8, 65, 16), (1, 3, 100003, 7), (9, 16, 4097, 48)])
def test_best_continuations(dtype, g, k, v, num):
    gen = torch.Generator().manual_seed(v + num)
    x = _logits((g, k, v), gen).to(dtype).to(DEV)
    scores = (-20 * torch.rand(g, k, generator=gen)).to(DEV)
    _check(x, scores, num)
    done = torch.rand(g, k, generator=gen).to(DEV) < 0.3
    _check(x, scores, num, done, v - 1)
    first = scores.clone()
    first[:, 1:] = -math.inf
    _check(x, first, num)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [7, 1001, 50021])
def test_equal_values_come_by_beam_and_token(dtype, v):
    gen = torch.Generator().manual_seed(v)
    few = torch.randint(-2, 3, (2, 1, v), generator=gen).to(dtype).to(DEV)
    x = few.expand(2, 5, v).contiguous()   # alike in every beam, at every alignment
    _check(x, torch.zeros(2, 5, device=DEV), min(64, 5 * v))
    _check(torch.zeros(1, 3, v, dtype=dtype, device=DEV), torch.zeros(1, 3, device=DEV), min(20, 3 * v))
    row = _logits((1, 1, v), gen).to(dtype).to(DEV).expand(1, 4, v).contiguous()
    _check(row, torch.full((1, 4), -3.25, device=DEV), min(30, 4 * v))


@pytest.mark.parametrize("num", [1, 9, 64])
def test_many_beams_alike(num):
    """More candidates than threads, all or most of them equal at the bound of the places."""
    gen = torch.Generator().manual_seed(num)
    for beams, v in ((64, 1001), (33, 70), (64, 20011)):
        row = torch.randint(-1, 2, (3, 1, v), generator=gen).half().to(DEV)
        x = row.expand(3, beams, v).contiguous()
        scores = torch.zeros(3, beams, device=DEV)
        scores[1, ::3] = -0.5
        scores[2] = (-torch.rand(beams, generator=gen)).to(DEV)
        done = torch.rand(3, beams, generator=gen).to(DEV) < 0.7
        _check(x, scores, num)
        _check(x, scores, num, done, 5)
        x[0, 1:] = -math.inf
        scores[1, 2:] = -math.inf
        _check(x, scores, num, done, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1001, 32000, 50021])
def test_values_closer_than_32_bits_tell(dtype, v):
    """Beams of one row whose scores differ by a step of 32 bits: the better score first, each time."""
    gen = torch.Generator().manual_seed(v)
    x = _logits((1, 1, v), gen, 3.0).to(dtype).to(DEV).expand(3, 4, v).contiguous()
    up = np.nextafter(np.float32(-0.75), np.float32(0))
    down = np.nextafter(np.float32(-0.75), np.float32(-1))
    scores = torch.tensor([[-0.75, up, down, -0.75], [down, -0.75, up, up], [up, up, down, -0.75]],
                          device=DEV)
    got = _check(x, scores, 24)
    # (a beam's other tokens of the same logit come before the next beam's)
    assert got.parents[0][got.tokens[0] == got.tokens[0, 0]].tolist() == [1, 0, 3, 2]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [-math.inf, "lowest", -6e4, -3e9, -1e30])
def test_masked_vocabularies(dtype, low):
    if low == "lowest":
        low = torch.finfo(dtype).min
    elif low < torch.finfo(dtype).min and low > -math.inf:
        pytest.skip("beyond the type")
    gen = torch.Generator().manual_seed(11)
    g, k, v = 6, 4, 9001
    x = _logits((g, k, v), gen).to(dtype)
    mask = torch.rand(g, k, v, generator=gen) < 0.95
    mask[1, 2] = True                       # a beam without a possible token
    mask[2] = True                          # a group without one
    mask[3] = True
    mask[3, 1, 77] = mask[3, 3, 8000] = False
    mask[4, :, :100] = True
    x = x.masked_fill(mask, low).to(DEV)
    scores = (-5 * torch.rand(g, k, generator=gen)).to(DEV)
    for num in (1, 8, 40):
        _check(x, scores, num)
    done = torch.zeros(g, k, dtype=torch.bool, device=DEV)
    done[1, 2] = done[2, 3] = done[3, 0] = done[5] = True
    _check(x, scores, 12, done, 3)


def test_beams_that_are_impossible_or_at_their_end():
    gen = torch.Generator().manual_seed(12)
    x = _logits((6, 3, 40), gen).to(DEV)
    scores = -torch.rand(6, 3, generator=gen).to(DEV)
    scores[0] = -math.inf                       # nothing goes on: the first tokens of the first beam
    scores[1, 0] = scores[1, 2] = -math.inf
    done = torch.zeros(6, 3, dtype=torch.bool, device=DEV)
    done[2] = True                              # three candidates, then impossible ones
    done[3, 0] = True
    done[4] = True
    scores[4, 1] = -math.inf
    x[5, 1] = -math.inf
    for num in (3, 10, 64):
        got = _check(x, scores, num, done, 2)
    assert got.tokens[0, :6].tolist() == [0, 1, 2, 3, 4, 5] and (got.parents[0, :40] == 0).all()
    # behind three possible ones: all tokens of the beams but the pad
    assert sorted(got.tokens[2, :3].tolist()) == [2, 2, 2] and got.tokens[2, 3:6].tolist() == [0, 1, 3]
    _check(x[:, :1, :2].contiguous(), scores[:, :1].contiguous(), 2, done[:, :1].contiguous(), 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_numbers(dtype):
    gen = torch.Generator().manual_seed(13)
    x = _logits((8, 3, 2049), gen).to(dtype).to(DEV)
    scores = -torch.rand(8, 3, generator=gen).to(DEV)
    done = torch.zeros(8, 3, dtype=torch.bool, device=DEV)
    x[0, 1, 700] = math.nan
    x[1, 2, 0] = math.inf
    scores[2, 0] = math.nan
    scores[3, 2] = math.inf
    x[4, 0, 5], done[4, 0] = math.nan, True     # not read
    x[5, 1, 5], scores[5, 1] = math.nan, -math.inf
    x[6, 0, 9] = x[6, 2, 9] = math.nan
    scores[7, 1], done[7, 1] = math.nan, True
    for num in (2, 9):
        _check(x, scores, num, done, 6)
    _check(x[..., :2].contiguous(), scores, 6, done, 1)


def test_logits_of_large_magnitude():
    gen = torch.Generator().manual_seed(14)
    x = _logits((4, 3, 5000), gen)
    x[0] += 1e6
    x[1] *= 1e7
    x[2] = x[2] * 1e30 - 1e31
    x[3, 1] = -2e9
    _check(x.to(DEV), -torch.rand(4, 3, generator=gen).to(DEV), 9)
    x = torch.randn(2, 3, 5000, generator=gen) * 1e-30   # differences that no sum can hold
    x[:, :, 4000:] = 3 * torch.arange(1000)[None, None] % 17
    _check(x.to(DEV), -torch.rand(2, 3, generator=gen).to(DEV), 9)


def test_rows_in_rising_order_and_long_ones():
    gen = torch.Generator().manual_seed(15)
    for v in (70000, 128256):
        x = torch.sort(_logits((1, 2, v), gen), -1)[0].to(DEV)
        for y in (x, x.flip(-1).contiguous(), x.half(), x.bfloat16()):
            _check(y, torch.tensor([[-1.0, -1.5]], device=DEV), 20)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_native_calls(dtype):
    gen = torch.Generator().manual_seed(16)
    base = _logits((4, 6, 3000), gen).to(dtype).to(DEV)
    scores = (-torch.rand(4, 6, generator=gen)).to(DEV)
    for x, s in ((base[..., 3:2500], scores), (base[1:, ::2, :999], scores[1:, ::2]),
                 (base.transpose(0, 1), scores.t()), (base[:, :1, 5:], scores[:, :1]),
                 (base[:2].transpose(1, 2).contiguous().transpose(1, 2), scores[:2])):
        got = _check(x, s, 7)
        want = S.beam_select(x, s, 7, None, 0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert beam_select(base, scores).tokens.shape == (4, 6)
    none = beam_select(base[:0], scores[:0], 3)
    assert none.scores.shape == none.tokens.shape == (0, 3)
    f = torch.compile(lambda t: beam_select(t, scores, 5).tokens * 2, backend="eager")
    assert torch.equal(f(base), beam_select(base, scores, 5).tokens * 2)


def test_a_small_workspace_gives_the_same():
    import ctypes

    gen = torch.Generator().manual_seed(17)
    g, k, v, num = 1, 3, 100003, 9
    x, scores = _logits((g, k, v), gen).to(DEV), (-torch.rand(g, k, generator=gen)).to(DEV)
    want = _check(x, scores, num)
    n = ctypes.c_size_t(0)
    lib = N.lib()
    assert lib.ojx_beam_select_workspace_bytes(g, k, v, num, 0, ctypes.byref(n)) == 0
    least = g * k * (16 + 8 * num)
    assert n.value > 2 * least
    out = [torch.empty(g, num, device=DEV), *(torch.empty(g, num, dtype=torch.int64, device=DEV)
                                              for _ in range(2))]
    for size in (least, 2 * least + 5, n.value):
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        assert lib.ojx_beam_select(N.ptr(x), v, g, k, v, 0, N.ptr(scores), 0, 0, num,
                                   *(N.ptr(t) for t in out), N.ptr(ws), size,
                                   N.stream_handle(DEV)) == 0
        assert torch.equal(out[1], want.parents) and torch.equal(out[2], want.tokens)
    assert lib.ojx_beam_select(N.ptr(x), v, g, k, v, 0, N.ptr(scores), 0, 0, num,
                               *(N.ptr(t) for t in out), N.ptr(ws), least - 1,
                               N.stream_handle(DEV)) == -1


def test_in_a_graph_and_on_a_stream():
    x = torch.randn(5, 4, 20000, device=DEV, dtype=torch.bfloat16)
    scores, done = torch.zeros(5, 4, device=DEV), torch.zeros(5, 4, dtype=torch.bool, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = beam_select(x, scores, 8, finished=done)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, beam_select(x, scores, 8, finished=done)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_select(x, scores, 8, finished=done)
    for i in range(4):
        x.copy_(torch.randn(5, 4, 20000, device=DEV) * 2)
        scores.copy_(-torch.rand(5, 4, device=DEV))
        done.copy_(torch.rand(5, 4, device=DEV) < 0.2)
        graph.replay()
        torch.cuda.synchronize()
        want = _check(x, scores, 8, done)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    x, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    d = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    for args, kw in (((x.double(), s, 2), {}), ((x[0], s, 2), {}), ((x, s.half(), 2), {}),
                     ((x, s[:1], 2), {}), ((x, s, 0), {}), ((x, s, 31), {}), ((x, s.cpu(), 2), {}),
                     ((x.cpu(), s.cpu(), 2), {}), ((x, s, 2), dict(finished=d.int())),
                     ((x, s, 2), dict(finished=d[:, :2])), ((x, s, 2), dict(finished=d, pad_id=10)),
                     ((x, s, 2), dict(finished=d, pad_id=-1)),
                     ((torch.zeros(1, 65, 10, device=DEV), torch.zeros(1, 65, device=DEV), 2), {}),
                     ((torch.zeros(1, 3, 100, device=DEV), s[:1], 65), {})):
        with pytest.raises(RuntimeError):
            beam_select(*args, **kw)
    with pytest.raises(RuntimeError):  # no gradient passes
        beam_select(x.clone().requires_grad_(True), s, 2).scores.sum().backward()
    assert ojasx_amd.BeamStep._fields == ("scores", "parents", "tokens")
