"""Gradients of rotations whose queries or keys need none: nothing is formed for those."""

import pytest
import torch

from ojasx_amd import rotary, serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
MIB = 1 << 20


def _both(q, k, pos, r, registered):
    if registered:
        return S.rotary(q, k, pos, r.rates, r.gain, r.interleaved, False)
    return rotary.rotate_qk(q, k, pos, r)


# (the registered op's formula is told by torch what requires a gradient, not what is asked for)
@pytest.mark.parametrize("registered,asked", [(False, "leaf"), (False, "input"), (True, "leaf")])
@pytest.mark.parametrize("frozen", ["q", "k"])
def test_nothing_for_what_needs_none(registered, frozen, asked):
    """The other's gradient is 16 MiB, which no call of a backward pass asks for: neither where the tensor
    is frozen nor where autograd.grad names the other alone."""
    t, d = 4096, 128
    r = rotary.rotation(d, device=DEV)
    pos = torch.arange(t, device=DEV)
    heads = {"q": 1, "k": 1, frozen: 16}
    x = {n: torch.randn(t, h, d, device=DEV, dtype=torch.bfloat16) for n, h in heads.items()}
    grads = {n: torch.randn_like(v) for n, v in x.items()}
    free = "k" if frozen == "q" else "q"
    x[free].requires_grad_(True)
    x[frozen].requires_grad_(asked == "input")
    y = dict(zip("qk", _both(x["q"], x["k"], pos, r, registered)))
    want = S.rotary(grads[free], None, pos, r.rates, r.gain, r.interleaved, True)[0]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got, = torch.autograd.grad([y["q"], y["k"]], [x[free]], [grads["q"], grads["k"]])
    assert torch.equal(got, want)
    assert torch.cuda.max_memory_allocated() - before < 4 * MIB  # the gradient itself is 1 MiB


def test_both_and_one_at_a_time():
    t, r = 50, rotary.rotation(64, device=DEV)
    pos = torch.arange(t, device=DEV)
    q, k = (torch.randn(t, h, 64, device=DEV, requires_grad=True) for h in (4, 2))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    back = lambda g: S.rotary(g, None, pos, r.rates, r.gain, r.interleaved, True)[0]  # noqa: E731
    y = rotary.rotate_qk(q, k, pos, r)
    for inputs, want in (([q, k], [back(gq), back(gk)]), ([k], [back(gk)]), ([q], [back(gq)])):
        got = torch.autograd.grad(y, inputs, [gq, gk], retain_graph=True)
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    # a gradient of the gradient, through one alone
    g = gk.clone().requires_grad_(True)
    got, = torch.autograd.grad(y, [k], [gq, g], create_graph=True)
    again, = torch.autograd.grad(got.sum(), [g])
    assert torch.equal(again, rotary.rotate(torch.ones_like(g), pos, r))
