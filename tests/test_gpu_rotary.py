"""Rotated positions against the definition in 64 bits, and their gradient."""

import math

import numpy as np
import pytest
import torch

import rotary_plain as P
from ojasx_amd import _native as N
from ojasx_amd import rotary, serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _check(got, x, r, positions, inverse=False):
    """`got` against x rotated: a rounding of the result beside the 32-bit products' error."""
    n = positions.cpu().numpy()
    want, bound = P.rotate(x.detach().cpu().double().numpy(), r.rates.cpu().numpy(), n, r.gain,
                           r.interleaved, inverse)
    # fp16 results under 2^-14 are multiples of 2^-24
    bound = bound * (1 + EPS[x.dtype]) + EPS[x.dtype] * np.abs(want) + \
        (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    assert got.dtype == x.dtype and got.shape == x.shape
    err = np.abs(got.detach().cpu().double().numpy() - want)
    assert (err <= bound).all(), float((err - bound).max())
    rot = 2 * r.rates.numel()
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("d,rot,hq,hkv,tokens", [
    (128, 128, 32, 8, 1), (128, 128, 32, 8, 65), (80, 32, 20, 20, 7), (80, 40, 5, 1, 33),
    (64, 64, 1, 1, 1000), (100, 100, 3, 1, 9), (100, 50, 3, 1, 9), (33, 2, 2, 1, 5), (7, 6, 1, 2, 5),
    (2, 2, 1, 1, 3), (256, 64, 9, 3, 17), (192, 190, 4, 2, 11), (72, 24, 7, 0, 130),
    (1024, 512, 2, 1, 3)])
def test_rotated_heads(dtype, interleaved, d, rot, hq, hkv, tokens):
    g = torch.Generator().manual_seed(d + tokens)
    x = (torch.randn(tokens, hq + hkv, d, generator=g) * 3).to(dtype).to(DEV)
    r = rotary.rotation(rot, interleaved=interleaved, device=DEV)._replace(gain=1.37)
    pos = torch.randint(0, 100000, (tokens,), generator=g, dtype=torch.int32).to(DEV)
    q, k = x[:, :hq], x[:, hq:]
    if hkv:
        a, b = rotary.rotate_qk(q, k, pos, r)
        _check(b, k, r, pos)
        assert torch.equal(rotary.rotate(k, pos.long(), r), b)
    else:
        a = rotary.rotate(q, pos, r)
    _check(a, q, r, pos)


def test_far_and_negative_positions():
    pos = torch.tensor([0, 1, -1, -7, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 3, 2 ** 62, -2 ** 62 - 5],
                       device=DEV)
    x = torch.randn(pos.numel(), 3, 64, device=DEV)
    r = rotary.rotation(64, device=DEV)
    _check(rotary.rotate(x, pos, r), x, r, pos)
    near = pos[:6].int()
    assert torch.equal(rotary.rotate(x[:6], near, r), rotary.rotate(x[:6], near.long(), r))
    # the angle itself, by its definition in 64 bits: 10^7 * f is known to 2^-30
    far = torch.tensor([9999991], device=DEV)
    y = rotary.rotate(torch.cat([torch.ones(32), torch.zeros(32)]).to(DEV)[None, None], far, r)
    f = torch.tensor(rotary.frequencies(64)[0], dtype=torch.float64) * far.item()
    assert (y[0, 0, :32].cpu().double() - f.cos()).abs().max() < 2.0 ** -21
    assert (y[0, 0, 32:].cpu().double() - f.sin()).abs().max() < 2.0 ** -21


def test_scaled_rotations():
    x = torch.randn(40, 2, 64, device=DEV)
    pos = torch.arange(40, device=DEV, dtype=torch.int32) * 997
    for scaling in ({"kind": "linear", "factor": 4}, {"kind": "base", "factor": 8},
                    {"kind": "ramp", "factor": 16, "length": 4096},
                    {"kind": "wavelength", "factor": 8, "length": 4096},
                    {"kind": "list", "factors": list(range(1, 33)), "gain": 1.2}):
        r = rotary.rotation(64, scaling=scaling, device=DEV)
        _check(rotary.rotate(x, pos, r), x, r, pos)


@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_are_taken_as_they_lie(dtype, interleaved):
    g = torch.Generator().manual_seed(5)
    b, s, h, d = 3, 37, 4, 96
    r = rotary.rotation(48, interleaved=interleaved, device=DEV)
    pos = torch.randint(0, 5000, (b, s), generator=g).to(DEV)
    base = torch.randn(b, s, 3 * h * d + 8, generator=g).to(dtype).to(DEV)
    parts = base[..., 3:3 + 3 * h * d].unflatten(-1, (3 * h, d))   # off the 16-byte grid
    for x in (base[..., :h * d].unflatten(-1, (h, d)),             # part of a product's output
              parts[..., h:2 * h, :], parts[:, ::2, ::3],           # holes over tokens and heads
              torch.randn(b, h, s, d, generator=g).to(dtype).to(DEV).transpose(1, 2),
              base[:, :, :d * h].unflatten(-1, (d, h)).transpose(2, 3),  # heads' elements apart
              base[:1, :, :h * d].unflatten(-1, (h, d)).expand(b, s, h, d)):
        p = pos[:, :x.shape[1]]
        for q in (p, p[0], p.t().contiguous().t(), p[0].int()):
            y = rotary.rotate(x, q, r)
            _check(y, x, r, q.expand(x.shape[:2]))
        a, c = rotary.rotate_qk(x, x[..., :1, :], p, r)
        assert torch.equal(a, rotary.rotate(x, p, r)) and torch.equal(c, a[..., :1, :])
        want = S.rotary(x, x[..., :1, :], p, r.rates, 1.0, interleaved, False)
        assert torch.equal(a, want[0]) and torch.equal(c, want[1])
        assert a.stride() == want[0].stride()


@pytest.mark.parametrize("dtype", list(EPS))
def test_heads_that_overlap(dtype):
    """Windows of one tensor: heads, or tokens, that share elements."""
    flat = torch.randn(5, 40, device=DEV).to(dtype)
    r = rotary.rotation(16, device=DEV)
    pos = torch.arange(5, device=DEV) * 1001
    few = flat[:, :18].unfold(1, 16, 1)
    assert few.shape == (5, 3, 16) and few.stride()[1:] == (1, 1)
    many = flat.unfold(1, 16, 1)
    along = flat[0, :20].unfold(0, 16, 1)[:, None]
    across = flat.flatten()[:60].view(20, 3).unfold(0, 16, 1)
    alike = flat[:1, None, :16].expand(5, 3, 16)
    for x in (few, many, along, across, alike):
        got = rotary.rotate(x, pos, r)
        assert got.stride(-1) == 1
        _check(got, x, r, pos)
        assert torch.equal(S.rotary(x, None, pos, r.rates, r.gain, False, False)[0], got)
        a, b = rotary.rotate_qk(x, few, pos, r)
        _check(a, x, r, pos)
        _check(b, few, r, pos)
    base = flat.clone().requires_grad_()
    rotary.rotate(base.unfold(1, 16, 1)[:, :3], pos, r).sum().backward()
    other = flat.clone().requires_grad_()
    rotary.rotate(other.unfold(1, 16, 1)[:, :3].contiguous(), pos, r).sum().backward()
    # the heads' parts may be added in another order: 3 terms
    assert (base.grad - other.grad).abs().max() <= 4 * EPS[dtype] * 6


def test_what_is_not_rotated_stays():
    x = torch.randn(4, 2, 40, device=DEV, dtype=torch.float16)
    x[..., 20:] = torch.tensor([math.nan, math.inf, -math.inf, 65504.0] * 5)
    pos = torch.arange(4, device=DEV)
    y = rotary.rotate(x, pos, rotary.rotation(20, device=DEV))
    assert torch.equal(y[..., 20:].view(torch.int16), x[..., 20:].view(torch.int16))
    x = torch.randn(2, 1, 8, device=DEV)
    x[0, 0, 1] = math.inf
    y = rotary.rotate(x, pos[:2] + 1, rotary.rotation(8, device=DEV))
    assert not torch.isfinite(y[0, 0, [1, 5]]).any() and torch.isfinite(y[0, 0, [0, 2, 3, 4, 6, 7]]).all()
    assert torch.isfinite(y[1]).all()


def test_no_tokens():
    r = rotary.rotation(64, device=DEV)
    for shape in ((0, 4, 64), (2, 0, 4, 64), (0, 5, 4, 64)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = rotary.rotate(x, torch.zeros(shape[:-2], dtype=torch.int32, device=DEV), r)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", list(EPS))
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(dtype, interleaved):
    g = torch.Generator().manual_seed(9)
    b, s, d = 2, 45, 80
    r = rotary.rotation(40, interleaved=interleaved, device=DEV)._replace(gain=1.3)
    pos = torch.randint(0, 30000, (b, s), generator=g).to(DEV)
    qkv = torch.randn(b, s, 8, d, generator=g).to(dtype).to(DEV).requires_grad_(True)
    gq, gk = (torch.randn(b, s, h, d, generator=g).to(dtype).to(DEV) for h in (5, 2))
    q, k = rotary.rotate_qk(qkv[..., :5, :], qkv[..., 5:7, :], pos, r)
    torch.autograd.backward([q, k], [gq, gk])
    _check(qkv.grad[..., :5, :], gq, r, pos, inverse=True)
    _check(qkv.grad[..., 5:7, :], gk, r, pos, inverse=True)
    assert (qkv.grad[..., 7, :] == 0).all()
    if dtype == torch.float32:
        # against differences: the map is linear, so those of any step are its product with v
        v = torch.randn(qkv.shape, generator=g).to(DEV)
        with torch.no_grad():
            a, c = rotary.rotate_qk((qkv + v)[..., :5, :], (qkv + v)[..., 5:7, :], pos, r)
            terms = torch.cat([((a - q).double() * gq).flatten(), ((c - k).double() * gk).flatten()])
            got = (qkv.grad.double() * v).sum()
        # sums of 50400 products with 32-bit values each off by 2^-20 of about 4 * 3
        assert abs(terms.sum() - got) < 50400 ** 0.5 * 12 * 2.0 ** -20 * 4


def test_in_autograd():
    """The recorded call against the registered op's formula, as autograd meets it."""
    r = rotary.rotation(16, device=DEV)
    pos = torch.arange(6, device=DEV) * 31
    base = torch.randn(6, 3, 24, device=DEV)

    def op(x, y=None):
        out = S.rotary(x, y, pos, r.rates, r.gain, r.interleaved, False)
        return out[0] if y is None else out

    def both(use):
        grads = []
        for one, two in ((lambda x: rotary.rotate(x, pos, r), lambda x, y: rotary.rotate_qk(x, y, pos, r)),
                         (op, op)):
            leaf = base.clone().requires_grad_(True)
            use(leaf, one, two)
            grads.append(leaf.grad)
        assert torch.equal(*grads) and grads[0].abs().max() > 0

    both(lambda t, f, g: f(t).sum().backward())                       # an expanded gradient
    both(lambda t, f, g: f(t)[:, ::2].square().sum().backward())
    both(lambda t, f, g: g(t, t[:, :1])[1].square().sum().backward())  # keys alone
    both(lambda t, f, g: g(t.detach(), t)[1].square().sum().backward())
    both(lambda t, f, g: sum(x.square().sum() for x in g(t, 2 * t)).backward())
    both(lambda t, f, g: f(t.transpose(0, 1).contiguous().transpose(0, 1)).square().sum().backward())
    both(lambda t, f, g: torch.utils.checkpoint.checkpoint(
        lambda u: f(u).square().sum(), t, use_reentrant=False).backward())

    def again(t, f, g):  # a gradient's gradient
        d, = torch.autograd.grad(f(t).pow(3).sum(), [t], create_graph=True)
        d.square().sum().backward()
    both(again)

    def twice(t, f, g):
        y = f(t).square().sum()
        y.backward(retain_graph=True)
        y.backward()
    both(twice)
    leaf = base.clone().requires_grad_(True)
    assert not rotary.rotate(leaf.detach(), pos, r).requires_grad
    with torch.no_grad():
        assert not rotary.rotate(leaf, pos, r).requires_grad


def test_calls_that_are_not_plain():
    r = rotary.rotation(16, device=DEV)
    pos = torch.arange(6, device=DEV)
    x = torch.randn(6, 3, 24, device=DEV)
    rest = (pos, r.rates, 1.0, False, False)
    assert N.eager().rotary(x.clone().requires_grad_(True), None, *rest) is None
    assert N.eager().rotary(x.double(), None, *rest) is None
    assert N.eager().rotary(x.transpose(1, 2).contiguous().transpose(1, 2), None, *rest) is None
    for args in ((x.double(), pos, r), (x[0], pos, r), (x, pos[:5], r), (x, pos.float(), r),
                 (x, pos, rotary.rotation(26, device=DEV)), (x, pos.cpu(), r),
                 (x, pos, rotary.rotation(16, device="cpu"))):
        with pytest.raises(RuntimeError):
            rotary.rotate(*args)
    with pytest.raises(RuntimeError):
        rotary.rotate_qk(x, x.half(), pos, r)
    # a rotation put together by hand
    by_hand = rotary.Rotation(r.rates, 2, 1)
    _check(rotary.rotate(x, pos, by_hand), x, by_hand, pos)
    f = torch.compile(lambda t: rotary.rotate(t, pos, r) * 2, backend="eager")
    assert torch.equal(f(x), rotary.rotate(x, pos, r) * 2)


def test_streams_and_graphs():
    r = rotary.rotation(128, device=DEV)
    x = torch.randn(50, 12, 128, device=DEV, dtype=torch.bfloat16)
    gy = torch.randn(50, 12, 128, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(50, device=DEV, dtype=torch.int32)
    leaf = x.clone().requires_grad_(True)

    def step():
        q, k = rotary.rotate_qk(leaf[:, :8], leaf[:, 8:], pos, r)
        g, = torch.autograd.grad([q, k], [leaf], [gy[:, :8], gy[:, 8:]])
        return q.detach(), k.detach(), g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # nothing of its graph is kept while another is captured
        first = step()[2]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(torch.randn(50, 12, 128, device=DEV))
        pos.copy_(torch.randint(0, 100000, (50,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
        assert not torch.equal(kept[2], first)
