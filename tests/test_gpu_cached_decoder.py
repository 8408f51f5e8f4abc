"""The example decoder: cache, attention and log probabilities run together.

In float32, against the same decoder with the cache's rules, the attention and the log
probabilities in plain Python and 64-bit arithmetic.
"""

import importlib.util
import os

import numpy as np
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def _example():
    path = os.path.join(os.path.dirname(HERE), "ojasx-open-source-cuda_amd", "examples",
                        "cached_decoder.py")
    spec = importlib.util.spec_from_file_location("cached_decoder", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class PlainCache:
    """KV8Cache's rules on the CPU."""

    def __init__(self, blocks, heads, dim, block):
        self.block = block
        self.k, self.v = (np.zeros((blocks, heads, block, P.stored(dim)), np.int64)
                          for _ in range(2))
        self.ks, self.vs = (np.zeros((blocks, heads), np.float32) for _ in range(2))

    def append(self, k, v, slots):
        s = slots.tolist()
        P.append(self.k, self.ks, k.cpu().numpy(), s, self.block)
        P.append(self.v, self.vs, v.cpu().numpy(), s, self.block)

    def attention(self, q, tables, lens, starts, **_):
        out = P.attention(q.cpu().double().numpy(), self.k, self.v, self.ks, self.vs,
                          tables.tolist(), lens.tolist(), starts.tolist(), q.shape[-1] ** -0.5, 0,
                          self.block)[0]
        return torch.from_numpy(out).to(q)


def test_answers_match_the_plain_decoder():
    ex = _example()
    model = ex.Decoder(layers=2, hidden=128, heads=6, kv_heads=2, head_dim=48, vocabulary=333,
                       dtype=torch.float32)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 333, (n,), generator=gen).tolist() for n in (1, 19, 5, 40)]
    tokens, lp, prompt_lp, states, batch, caches = ex.answer(model, prompts, 9, num_blocks=24)
    assert batch.lens.tolist() == [9, 27, 13, 48]
    assert batch.num_free.item() == 24 - (1 + 2 + 1 + 3)
    used = [b for r, n in zip(batch.tables.tolist(), (1, 2, 1, 3)) for b in r[:n]]
    assert len(set(used)) == 7

    # Same tokens through the plain cache, so every step's state can be compared.  Both sides are
    # 32-bit sums of at most 512 terms of order 1 outside the attention: 1e-5 in a state of order
    # 1.  Such a difference can also turn a key's or value's rounding at a half: one code of 127
    # off, in one element of one of the visible tokens, so one term of a score or of an output is
    # off by 1/127 of the block's largest, about 4/127; times a weight of order 1 / tokens and a
    # product of order 48^-1/2: below 5e-3 for the shortest rows.
    device = tokens.device
    plain = [PlainCache(24, 2, 48, 16) for _ in caches]
    again = ex.Requests(4, 49, 24, 16, device)
    with torch.no_grad():
        ids = torch.tensor([t for p in prompts for t in p], device=device)
        plan = again.step(torch.tensor([len(p) for p in prompts], dtype=torch.int32,
                                       device=device), len(ids))
        h = model.hidden(ids, plan, again.tables, plain)
        logits = model.head(h).double().cpu()
        want = torch.log_softmax(logits, -1)
        follow = [t for p in prompts for t in (*p[1:], -1)]
        for row, (t, got) in enumerate(zip(follow, prompt_lp.tolist())):
            assert abs(got - (want[row, t].item() if t >= 0 else 0.0)) < 5e-3
        last = h[plan.query_starts[1:].long() - 1]
        for i in range(9):
            torch.testing.assert_close(states[:, i], last, rtol=0, atol=5e-3)
            want = torch.log_softmax(model.head(last).double().cpu(), -1)
            at = want.gather(1, tokens[:, i:i + 1].cpu())[:, 0]
            torch.testing.assert_close(lp[:, i].cpu().double(), at, rtol=0, atol=5e-3)
            assert (want.max(1).values - at).max() < 1e-2  # the chosen one is the most likely
            if i < 8:
                plan = again.step(torch.ones(4, dtype=torch.int32, device=device), 4)
                last = model.hidden(tokens[:, i], plan, again.tables, plain)


def test_policy_steps_raise_the_better_answers():
    ex = _example()
    model = ex.Decoder(layers=1, dtype=torch.float32)
    prompts = [[1, 2, 3], [4], [5, 6], list(range(30))]
    tokens, lp, _, states, _, _ = ex.answer(model, prompts, 6)
    rewards = torch.tensor([1.0, 0.0, 1.0, 0.0], device=tokens.device)
    losses = ex.reinforce(model, states, tokens, lp, rewards, steps=6, rate=0.05,
                          entropy_weight=0.0)
    assert torch.isfinite(losses).all()
    assert losses[0].abs() < 1e-4       # ratios of 1 and gains that sum to zero
    assert losses[-1] < losses[0]       # and falls from there
    with torch.no_grad():
        change = (ex.token_logprobs(model.head(states), tokens).logprob - lp).mean(1)
    assert change[[0, 2]].mean() > change[[1, 3]].mean()


def test_command_prints(capsys):
    _example().main()
    out = capsys.readouterr().out
    left = 64 - sum(-(-(n + 23) // 16) for n in (1, 37, 16, 120))  # the last token is not cached
    assert f"blocks left {left}" in out and "losses" in out
