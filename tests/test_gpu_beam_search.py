"""Beam search of the example decoder: rotated appends, attention, selection, reordered caches and
copied blocks run together."""

import numpy as np
import pytest
import torch

import beam_plain as P
import kv8_plain
from ojasx_amd import kv8
from test_gpu_cached_decoder import _example

pytestmark = pytest.mark.gpu

PROMPTS = (1, 19, 5, 40, 16)


def _search(dtype, beams, new, end, block_size=16):
    ex = _example()
    model = ex.Decoder(layers=2, hidden=128, heads=6, kv_heads=2, head_dim=48, vocabulary=333, dtype=dtype)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 333, (n,), generator=gen).tolist() for n in PROMPTS]
    steps = []
    out = ex.beam_answer(model, prompts, beams, new, end, num_blocks=200, block_size=block_size,
                         watch=lambda *a: steps.append(a))
    return ex, model, prompts, steps, out


@pytest.mark.parametrize("dtype,beams,block", [(torch.float32, 4, 16), (torch.bfloat16, 3, 16),
                                               (torch.float16, 1, 64), (torch.bfloat16, 8, 32)])
def test_every_choice_is_the_best(dtype, beams, block):
    _, _, _, steps, (answers, scores, batch, caches) = _search(dtype, beams, 14, end=5, block_size=block)
    assert len(steps) == 14 and answers.shape == (5, beams, 14)
    for logits, before, done, best in steps:
        want = P.select(logits.float().cpu().numpy(), before.cpu().numpy(), beams, done.cpu().numpy(), 5)
        assert np.array_equal(best.parents.cpu().numpy(), want[1])
        assert np.array_equal(best.tokens.cpu().numpy(), want[2])
        np.testing.assert_allclose(best.scores.cpu().numpy(), want[0], rtol=2.0 ** -23, atol=2.0 ** -20)
    # blocks: what the tables hold and the stack are all blocks, once each
    lens = batch.lens.tolist()
    assert lens == [n + 13 for n in PROMPTS for _ in range(beams)]
    held = {b for row, n in zip(batch.tables.tolist(), lens) for b in row[:-(-n // block)]}
    left = batch.num_free.item()
    stack = batch.free[:left].tolist()
    assert len(stack) == left and held | set(stack) == set(range(200)) and not held & set(stack)
    # begun blocks are each one row's own
    begun = [row[n // block] for row, n in zip(batch.tables.tolist(), lens) if n % block]
    assert len(set(begun)) == len(begun)
    batch.go_on(torch.full((3,), -1, device=batch.lens.device), 200, caches)
    assert batch.num_free.item() == 200 and sorted(batch.free.tolist()) == list(range(200))
    assert batch.lens.tolist() == [0, 0, 0] and (batch.tables == -1).all()


def test_shared_caches_hold_what_own_ones_would():
    """The answers once more, each in blocks of its own from the prompt on: the same codes, states and
    log probabilities.

    Rows of a batch of one size go through the same products, but the prompts' rows need not: sums of
    at most 512 terms of order 1 in another order, 1e-5, which can turn a code's rounding (the bound
    and its reason are those of the greedy answers' test)."""
    beams, new = 4, 14
    ex, model, prompts, _, (answers, scores, batch, caches) = _search(torch.float32, beams, new, end=400 % 333)
    rows = [p for p in prompts for _ in range(beams)]
    lens = [len(p) for p in rows]
    device = answers.device
    own = ex.Requests(len(rows), max(lens) + new, 400, 16, device)
    again = model.caches(400, 16)
    tokens = torch.tensor([t for p in rows for t in p], device=device)
    flat = answers.flatten(0, 1)
    total = torch.zeros(len(rows), dtype=torch.float64)
    done = torch.zeros(len(rows), dtype=torch.bool)
    with torch.no_grad():
        plan = own.step(torch.tensor(lens, dtype=torch.int32, device=device), len(tokens))
        h = model.hidden(tokens, plan, own.tables, again, True)[plan.query_starts[1:].long() - 1]
        for i in range(new):
            lp = torch.log_softmax(model.head(h).double(), -1).gather(1, flat[:, i:i + 1])[:, 0].cpu()
            total += torch.where(done, 0.0, lp)
            done |= flat[:, i].cpu() == 400 % 333
            if i + 1 < new:
                plan = own.step(torch.ones(len(rows), dtype=torch.int32, device=device), len(rows))
                h = model.hidden(flat[:, i], plan, own.tables, again, True)
    torch.testing.assert_close(total, scores.flatten().double().cpu(), rtol=0, atol=5e-3 * new)
    for a, b in zip(caches, again):
        for x, y, xs, ys in zip(kv8_plain.codes_of(a), kv8_plain.codes_of(b), a.scales.unbind(-1),
                                b.scales.unbind(-1)):
            off = count = 0
            for r, n in enumerate(own.lens.tolist()):
                for j in range(-(-n // 16)):
                    p, q = batch.tables[r, j].item(), own.tables[r, j].item()
                    k = min(16, n - 16 * j)
                    torch.testing.assert_close(xs[p], ys[q], rtol=1e-4, atol=0)
                    d = np.abs(x[p][:, :k] - y[q][:, :k])
                    assert d.max() <= 1
                    off, count = off + (d > 0).sum(), count + d.size
            assert off < count / 500


def test_one_prompt_for_many():
    """Several answers of one prompt: its rows share the prompt's blocks, and part where they differ."""
    dev = torch.device("cuda:0")
    c = kv8.KV8Cache(12, 1, 64, 16, dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    x = torch.randn(40, 1, 64, device=dev, dtype=torch.bfloat16)
    p = kv8.plan(i32([0]), i32([40]), (tables := torch.zeros(1, 4, dtype=torch.int32, device=dev)),
                 torch.arange(12, dtype=torch.int32, device=dev), i32([12]), 16, 40)
    c.append(x, x, p.slots)
    r = kv8.reorder(torch.tensor([0, 0, 0], device=dev), p.seq_lens, tables,
                    torch.arange(12, dtype=torch.int32, device=dev), p.num_free, 16, 12)
    kv8.copy_blocks([c], r.sources, r.targets)
    assert r.block_tables[:, :3].tolist() == [[11, 10, 9], [11, 10, 8], [11, 10, 7]]
    q = torch.randn(3, 2, 64, device=dev, dtype=torch.bfloat16)
    same = c.attention(q[:1].expand(3, -1, -1), r.block_tables, r.seq_lens)
    assert torch.equal(same[0], same[1]) and torch.equal(same[0], same[2])
    y = torch.randn(3, 1, 64, device=dev, dtype=torch.bfloat16)
    p = kv8.plan(r.seq_lens, i32([1, 1, 1]), r.block_tables, r.free_blocks, r.num_free, 16, 3)
    c.append(y, y, p.slots)
    apart = c.attention(q, r.block_tables, p.seq_lens)
    for i in range(3):
        own = kv8.KV8Cache(3, 1, 64, 16, dev)
        own.append(x, x, torch.arange(40, device=dev))
        own.append(y[i:i + 1], y[i:i + 1], torch.tensor([40], device=dev))
        assert torch.equal(apart[i:i + 1], own.attention(q[i:i + 1], i32([[0, 1, 2, -1]]), i32([41]),
                                                         max_seq_len=64))


def test_command_prints_beams(capsys):
    _example().main()
    out = capsys.readouterr().out
    assert "best of four beams" in out and "blocks given back 256" in out
