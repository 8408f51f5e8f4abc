"""Token log probabilities and their gradient on the GPU against float64.

Bounds: fp32 sums of V terms over at least 64 lanes are off by (V / 64 + 32) roundings at most,
the exponentials by the rounding of their argument (its size times 2^-24) and 2 ulp of their own.
"""

import math

import numpy as np
import pytest
import torch

import kv8_plain as P
import ojasx_amd
from ojasx_amd import serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
ULP = 2.0 ** -23
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(rows, v, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, v, generator=g) * spread).to(dtype)


def _check(x, ids, top, view=None):
    """x on the CPU in its dtype; view: how it is given on the GPU."""
    xd = (view or (lambda t: t.to(DEV)))(x)
    got = ojasx_amd.token_logprobs(xd, torch.tensor(ids, dtype=torch.int64, device=DEV), top_k=top)
    x64 = x.double().numpy()
    lp, h, lse, best, order, _ = P.logprobs(x64, ids, top)
    v = x.shape[1]
    fin = np.where(np.isfinite(x64), x64, np.nan)
    with np.errstate(invalid="ignore"):
        import warnings
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            big = np.nan_to_num(np.nanmax(np.abs(fin), 1)) + 20
    tol = ULP * (big + v / 64 + 32)

    def near(a, b, t):
        a = a.double().cpu().numpy()
        same = (a == b) | (np.abs(a - np.where(np.isfinite(b), b, 0)) <= t)
        assert (same & (np.isfinite(a) == np.isfinite(b))).all()

    near(got.logprob, lp, tol)
    near(got.lse, lse, tol)
    near(got.entropy, h, tol * (1 + np.log(v)))
    assert got.top_ids.dtype == torch.int64 and got.top_ids.shape == (x.shape[0], top)
    assert np.array_equal(got.top_ids.cpu().numpy(), order)
    near(got.top_logprobs, best, tol[:, None])
    return got


def _ids(rows, v, seed=0):
    return np.random.RandomState(seed).randint(0, v, rows).tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v,top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 65, 64), (7, 255, 3),
    (3, 1000, 20), (2, 4097, 8), (9, 8192, 1), (2, 32003, 64), (1, 128256, 8), (300, 515, 5),
    (1100, 2048, 0), (3, 50021, 20), (1, 200001, 0)])
def test_values(dtype, rows, v, top):
    _check(_logits(rows, v, dtype, rows + v), _ids(rows, v), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [7, 64, 3000, 70001])
def test_equal_logits_come_by_rising_token(dtype, v):
    top = min(v, 64)
    _check(torch.zeros(2, v, dtype=dtype), _ids(2, v), top)
    x = _logits(6, v, dtype, v).round()  # few distinct values
    x[4] = torch.where(torch.rand(v) < 0.5, 0.0, -0.0)
    x[5] = torch.arange(v) % 3
    _check(x, _ids(6, v), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 300, 20000])
def test_ordered_rows(dtype, v):
    # the largest together at one end, or in one lane's share
    x = torch.zeros(4, v)
    x[0] = torch.linspace(-5, 5, v)
    x[1] = x[0].flip(0)
    x[2, : v // 8 + 1] = 7
    x[3, ::256] = torch.linspace(1, 2, len(x[3, ::256]))
    _check(x.to(dtype), [0, v - 1, v // 2, 0], min(v, 40))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [6, 515, 40000])
def test_masked_rows(dtype, v):
    x = _logits(7, v, dtype, v)
    x[0] = -math.inf                                # nothing left
    x[1, 1:] = -math.inf                            # one token left
    x[2, torch.rand(v) < 0.9] = -math.inf
    x[2, 3] = 1.0
    x[3] = torch.finfo(dtype).min                   # the type's lowest value everywhere
    x[4, : v - 2] = torch.finfo(dtype).min
    x[5, v // 2:] = -math.inf
    ids = [2, 0, 3, 1, v - 1, v - 1, -100]          # of them a masked one, one not asked for
    _check(x, ids, min(v, 30))
    _check(x, [v, -1, 2 ** 40, -2 ** 40, v + 7, 0, 1], 2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v,top", [(1, 2054, 20), (2, 70001, 64), (300, 4100, 5)])
def test_few_allowed_tokens(dtype, rows, v, top):
    # fewer logits than alternatives, at the ends, together and far apart; the others masked
    for low in (-math.inf, torch.finfo(dtype).min):
        x = torch.full((rows, v), low)
        x[0, [0, v // 2, v - 1]] = torch.tensor([1.0, 3.0, 2.0])
        if rows > 1:
            x[1, v - 3:] = 0.25
            x[2:, 7::v // 4] = 0.5
        _check(x.to(dtype), _ids(rows, v), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [2048, 9000])
def test_equal_logits_among_rising_and_falling_ones(dtype, v):
    # more candidates than are kept at a time, equal ones among them in both orders of place
    j = torch.arange(v)
    x = torch.stack([(j // 3 % 900).float(), (j // 64).float(), (j % 64).float(),
                     -(j // 5 % 700).float(), (j // 40 * 7 % 64).float()]) / 32
    _check(x.to(dtype), _ids(5, v), 64)
    _check(x.to(dtype), _ids(5, v), 33)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [9, 3000, 40000])
def test_nan_and_infinity(dtype, v):
    x = _logits(3, v, dtype, v)
    x[0, v - 1] = math.nan
    x[1, 4] = math.inf
    ids = torch.tensor([0, 4, 1], device=DEV)
    got = ojasx_amd.token_logprobs(x.to(DEV), ids, top_k=3)
    for t in (got.logprob, got.entropy, got.lse):
        assert t[:2].isnan().all() and not t[2].isnan()
    assert got.top_logprobs[:2].isnan().all() and not got.top_logprobs[2].isnan().any()
    assert got.top_ids[0, 0] == v - 1 and got.top_ids[1, 0] == 4


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_shapes_and_another_stream(dtype):
    x = _logits(6, 1003, dtype, 4)
    wide = torch.randn(6, 1500).to(dtype).to(DEV)

    def cut(at):
        def view(t):
            wide[:, at:at + 1003] = t.to(DEV)
            return wide[:, at:at + 1003]
        return view

    for at in (0, 1, 8, 497):
        _check(x, _ids(6, 1003), 7, cut(at))
    _check(x, _ids(6, 1003), 7, lambda t: t.t().contiguous().to(DEV).t())
    _check(x[:1].expand(6, -1), _ids(6, 1003), 7, lambda t: x[:1].to(DEV).expand(6, -1))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = _check(x, _ids(6, 1003), 7)
    torch.cuda.current_stream().wait_stream(side)
    b = ojasx_amd.token_logprobs(x.to(DEV).reshape(2, 3, 1003),
                                 torch.tensor(_ids(6, 1003), device=DEV).reshape(2, 3), top_k=7)
    for s, t in zip(a, b):
        assert torch.equal(s, t.reshape(s.shape)) and t.shape[:2] == (2, 3)
    none = ojasx_amd.token_logprobs(x.to(DEV)[:0], torch.zeros(0, dtype=torch.int64, device=DEV), 2)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 2)


# ------------------------------------------------------------------ gradient

def _grad_of(x, ids, top, grads, view=None):
    xd = (view or (lambda t: t.to(DEV)))(x).detach().requires_grad_(True)
    out = ojasx_amd.token_logprobs(xd, torch.tensor(ids, dtype=torch.int64, device=DEV), top_k=top)
    outs = [out.logprob, out.entropy, out.lse, out.top_logprobs]
    use = [(o, g.to(DEV)) for o, g in zip(outs, grads) if g is not None]
    return torch.autograd.grad([o for o, _ in use], [xd], [g for _, g in use])[0]


def _check_grad(x, ids, top, which="lhst", view=None):
    rows, v = x.shape
    g = torch.Generator().manual_seed(rows * v)
    grads = [torch.randn(rows, generator=g) if c in which else None for c in "lhs"]
    grads.append(torch.randn(rows, top, generator=g) if "t" in which and top else None)
    if all(t is None for t in grads):
        return
    got = _grad_of(x, ids, top, grads, view).double().cpu().numpy()
    x64 = x.double().numpy()
    lp, h, lse, best, order, logp = P.logprobs(x64, ids, top)
    p = np.exp(logp)
    logp = np.where(p > 0, logp, 0)
    gl, gh, gs, gt = (t.double().numpy() if t is not None else None for t in grads)
    want = np.zeros_like(x64)
    parts = np.zeros_like(x64)  # sums of |terms|
    for r in range(rows):
        terms = []
        if gl is not None and 0 <= ids[r] < v:
            one = np.zeros(v)
            one[ids[r]] = 1
            terms += [gl[r] * one, -gl[r] * p[r]]
        if gh is not None:
            terms += [-gh[r] * p[r] * logp[r], -gh[r] * p[r] * h[r]]
        if gs is not None:
            terms += [gs[r] * p[r]]
        if gt is not None:
            for i in range(top):
                one = np.zeros(v)
                one[order[r, i]] = 1
                terms += [gt[r, i] * one, -gt[r, i] * p[r]]
        for t in terms:
            want[r] += t
            parts[r] += np.abs(t)
    big = np.abs(logp) + 20
    bound = HALF_ULP[x.dtype] * np.abs(want) + parts * ULP * (2 * big + v / 32 + 64 + top) + 2.0 ** -25
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (3, 2, 2), (2, 63, 0), (5, 300, 64), (3, 4097, 5),
                                        (2, 32003, 20), (1, 128256, 0), (130, 515, 3)])
@pytest.mark.parametrize("which", ["l", "h", "lhst"])
def test_gradient(dtype, rows, v, top, which):
    ids = _ids(rows, v, 1)
    ids[0] = -100 if rows > 1 else ids[0]
    _check_grad(_logits(rows, v, dtype, v), ids, top, which)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_masked_rows_and_named_tokens(dtype):
    v = 700
    x = _logits(5, v, dtype, 9)
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, torch.rand(v) < 0.9] = -math.inf
    x[2, 3] = 1.0
    x[3] = torch.finfo(dtype).min
    x[4, 17] = 30  # the given token is the first alternative
    _check_grad(x, [2, 0, 3, 1, 17], 12)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_strided_rows(dtype):
    x = _logits(4, 501, dtype, 4)
    wide = torch.randn(4, 777).to(dtype).to(DEV)
    for at in (0, 3):
        def view(t, at=at):
            wide[:, at:at + 501] = t.to(DEV)
            return wide[:, at:at + 501]
        _check_grad(x, _ids(4, 501), 3, view=view)


def test_gradient_against_differences():
    rows, v, top = 6, 900, 5
    g = torch.Generator().manual_seed(2)
    # logits a tenth apart at least, so that a step keeps the alternatives' order
    x = torch.stack([torch.randperm(v, generator=g) for _ in range(rows)]).float() * 0.1 - 40
    ids = torch.tensor(_ids(rows, v), device=DEV)
    c = [torch.randn(rows, generator=g).to(DEV) for _ in range(3)] + \
        [torch.randn(rows, top, generator=g).to(DEV)]
    x = x.to(DEV).requires_grad_(True)

    def loss(t):
        out = ojasx_amd.token_logprobs(t, ids, top_k=top)
        vals = (out.logprob, out.entropy, out.lse, out.top_logprobs)
        return sum((a.double() * b.double()).sum() for a, b in zip(vals, c))

    grad, = torch.autograd.grad(loss(x), [x])
    step = 0.02  # differences: truncation step^2 of third derivatives (O(1)), rounding 1e-5 / step
    for i in range(4):
        e = torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        e = e / e.abs().amax()
        with torch.no_grad():
            slope = (loss(x + step * e) - loss(x - step * e)).item() / (2 * step)
        assert abs(slope - (grad.double() * e).sum().item()) <= 5e-3


def test_registered_op_and_compiled_call():
    x = _logits(3, 200, torch.float32, 1).to(DEV).requires_grad_(True)
    ids = torch.tensor([1, 2, 199], device=DEV)
    want = ojasx_amd.token_logprobs(x, ids, top_k=2)
    got = torch.ops.ojasx_e8t.token_logprobs(x, ids, 2)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    a, = torch.autograd.grad(want.logprob.sum() + want.entropy.sum(), [x])
    b, = torch.autograd.grad(got[0].sum() + got[1].sum(), [x])
    assert torch.equal(a, b)
    torch.library.opcheck(S.token_logprobs, (x.detach(), ids, 2),
                          test_utils=("test_schema", "test_faketensor"))


def test_rows_of_zero_gradient_are_zero_and_unused_results_cost_nothing():
    x = _logits(4, 100, torch.bfloat16, 1).to(DEV).requires_grad_(True)
    out = ojasx_amd.token_logprobs(x, torch.tensor([-1, 5, -1, 7], device=DEV))
    g, = torch.autograd.grad(out.logprob.sum(), [x])
    assert not g[0].any() and not g[2].any() and g[1].any()
