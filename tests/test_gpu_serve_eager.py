"""The cache's and token_logprobs' plain eager calls (native code) against the registered ops, and
the calls that have to take the registered op."""

import pytest
import torch
import torch.utils.checkpoint

import kv8_plain as P
import ojasx_amd
from ojasx_amd import _native as N
from ojasx_amd import kv8, serve_ops as S

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(seed=0):
    c = ojasx_amd.KV8Cache(20, 2, 96, 16, DEV)
    P.fill(c, torch.Generator().manual_seed(seed))
    return c


def test_plan_append_read_and_attention_match_the_ops():
    tables = torch.full((3, 6), -1, dtype=torch.int32, device=DEV)
    args = (_i32([0, 0, 0]), _i32([20, 1, 33]))
    rest = (_i32(list(range(20))), _i32([20]), 16, 54)
    other = tables.clone()
    version = tables._version
    a = kv8.plan(*args, tables, *rest)
    b = S.kv8_plan(*args, other, *rest)
    assert tables._version > version
    assert all(torch.equal(x, y) and x.dtype == y.dtype for x, y in zip(a, b))
    assert torch.equal(tables, other)
    c, d = _cache(), _cache()
    k, v = torch.randn(2, 54, 2, 96, device=DEV, dtype=torch.float16).unbind(0)
    version = c.k_codes._version
    c.append(k, v, a.slots)
    assert c.k_codes._version > version
    S.kv8_append(k, v, a.slots, d.k_codes, d.v_codes, d.scales)
    for x, y in ((c.k_codes, d.k_codes), (c.v_codes, d.v_codes), (c.scales, d.scales)):
        assert torch.equal(x, y)
    blocks = _i32([3, 19, -1])
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = c.read(blocks, dtype)
        want = S.kv8_read(c.k_codes, c.v_codes, c.scales, blocks, 96, dtype)
        assert all(torch.equal(x, y) and x.dtype == y.dtype for x, y in zip(got, want))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        q = torch.randn(54, 4, 96, device=DEV).to(dtype)
        for rows, starts, most in ((q, a.query_starts, 33), (q[:3], None, 1)):
            got, lse = c.attention(rows, tables, a.seq_lens, starts, return_lse=True, window=9)
            want = S.kv8_attention(rows, c.k_codes, c.v_codes, c.scales, tables, a.seq_lens, starts,
                                   96 ** -0.5, 9, most if starts is None else 54, 96, True)
            assert torch.equal(got, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("top", [0, 5])
def test_token_logprobs_match_the_op(top):
    ids = torch.tensor([[3, -1, 100], [7, 200, 0]], device=DEV)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = (torch.randn(2, 3, 201, device=DEV) * 3).to(dtype)
        want = S.token_logprobs(x, ids, top)
        got = ojasx_amd.token_logprobs(x, ids, top_k=top)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        grads = []
        for call in (ojasx_amd.token_logprobs, S.token_logprobs):
            leaf = x.clone().requires_grad_(True)
            out = call(leaf, ids, top)
            loss = out[0].sum() + 2 * out[1].sum() - out[2].mean() + out[3].sum()
            loss.backward()
            grads.append(leaf.grad)
        assert torch.equal(*grads)
        # only some results used; a leaf of another type behind a cast
        leaf = x.float().requires_grad_(True)
        ojasx_amd.token_logprobs(leaf.to(dtype), ids).entropy.sum().backward()
        assert leaf.grad.dtype == torch.float32 and torch.isfinite(leaf.grad).all()


def test_calls_that_are_not_plain():
    x = torch.randn(3, 50, device=DEV)
    ids = torch.tensor([1, 2, 3], device=DEV)
    assert N.eager().token_logprobs(x.t().contiguous().t(), ids, 2) is None
    assert N.eager().token_logprobs(x.clone().requires_grad_(True), ids, 2) is None
    assert N.eager().token_logprobs(x, ids.int(), 2) is None
    with pytest.raises(RuntimeError):
        ojasx_amd.token_logprobs(x, ids.int())
    with pytest.raises(RuntimeError):
        ojasx_amd.token_logprobs(x, ids, top_k=65)
    with pytest.raises(RuntimeError):
        ojasx_amd.token_logprobs(x.cpu(), ids.cpu())
    c = _cache()
    q = torch.randn(2, 4, 96, device=DEV, dtype=torch.bfloat16)
    tables, lens = _i32([[1, 2], [3, 4]]), _i32([20, 9])
    for bad in ((q.double(), tables, lens), (q[..., :20], tables, lens), (q, tables.long(), lens),
                (q, tables, lens[:1]), (q, tables, lens.cpu())):
        with pytest.raises(RuntimeError):
            c.attention(*bad)
    with pytest.raises(RuntimeError):  # no gradient passes the cache
        out = c.attention(q.clone().requires_grad_(True), tables, lens)
        out.float().sum().backward()
    # a double backward is refused, not wrong
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(ojasx_amd.token_logprobs(leaf, ids).logprob.sum(), [leaf],
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_recorded_logprobs_in_autograd():
    """The recorded call against the registered op's formula, as autograd meets it."""
    ids = torch.tensor([3, -1, 100], device=DEV)
    base = torch.randn(3, 300, device=DEV)

    def both(use):
        grads = []
        for call in (ojasx_amd.token_logprobs, S.token_logprobs):
            leaf = base.clone().requires_grad_(True)
            use(leaf, lambda t, k=4: call(t, ids, k))
            grads.append(leaf.grad)
        assert torch.equal(*grads) and grads[0].abs().max() > 0

    both(lambda t, f: f(t[:, :201])[0].sum().backward())                    # rows with a stride
    both(lambda t, f: f(t.t().contiguous().t())[1].sum().backward())        # laid out across
    both(lambda t, f: f(t)[3][:, ::2].sum().backward())                     # grads with holes
    both(lambda t, f: (f(t)[0].sum() + f(t * 2)[2].sum()).backward())       # twice in a graph
    both(lambda t, f: f(t)[0].backward(torch.ones(3, device=DEV).expand(3)))
    both(lambda t, f: torch.utils.checkpoint.checkpoint(
        lambda u: f(u)[0].sum(), t, use_reentrant=False).backward())

    def twice(t, f):
        y = f(t)[0].sum()
        y.backward(retain_graph=True)
        y.backward()
    both(twice)

    leaf = base.clone().requires_grad_(True)
    out = ojasx_amd.token_logprobs(leaf, ids, 4)
    assert out.logprob.requires_grad and not out.top_ids.requires_grad
    work = leaf * 1
    out = ojasx_amd.token_logprobs(work, ids)
    work.add_(1)  # what the gradient is formed from
    with pytest.raises(RuntimeError):
        out.logprob.sum().backward()
    out = ojasx_amd.token_logprobs(leaf.detach(), ids)
    assert not out.logprob.requires_grad
    with torch.no_grad():
        assert not ojasx_amd.token_logprobs(leaf, ids).logprob.requires_grad


def test_compiled_call_takes_the_op():
    x = torch.randn(3, 50, device=DEV)
    ids = torch.tensor([1, 2, 3], device=DEV)
    f = torch.compile(lambda t: ojasx_amd.token_logprobs(t, ids, top_k=2).entropy * 2,
                      backend="eager")
    assert torch.equal(f(x), ojasx_amd.token_logprobs(x, ids, top_k=2).entropy * 2)
