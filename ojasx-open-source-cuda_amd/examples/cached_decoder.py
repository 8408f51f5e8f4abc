"""A small decoder of packed linears that answers from an 8-bit cache, and learns from its answers.

    python ojasx-open-source-cuda_amd/examples/cached_decoder.py

Random weights, synthetic prompts of different lengths.  One batch goes through every operator
as a serving loop uses them: the cache's plan, append and attention in each step (a step holds
prompts, single tokens, or both), the prompts' own log probabilities, the most likely next token
with its log probability, a few steps of policy training of the head's adapter on the answers, and at
the end the prompts again by beam search, whose beams share their blocks and whose positions are
rotated on the way into the cache.  No step waits for the GPU: lengths, tables and tokens stay there.
"""

from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ojasx_amd import (E8LatticeLinear, KV8Cache, beam_select, kv8, rotary,  # noqa: E402
                       token_logprobs)


class Requests:
    """A batch's blocks: tables, lengths and the stack of free blocks, on the GPU."""

    def __init__(self, count: int, longest: int, num_blocks: int, block_size: int, device="cuda"):
        width = (longest + block_size - 1) // block_size
        self.longest, self.block_size = longest, block_size
        self.tables = torch.zeros(count, width, dtype=torch.int32, device=device)
        self.lens = torch.zeros(count, dtype=torch.int32, device=device)
        self.free = torch.arange(num_blocks, dtype=torch.int32, device=device)
        self.num_free = torch.tensor([num_blocks], dtype=torch.int32, device=device)

    def step(self, new_lens: torch.Tensor, num_tokens: int) -> kv8.KV8Plan:
        plan = kv8.plan(self.lens, new_lens, self.tables, self.free, self.num_free,
                        self.block_size, num_tokens)
        self.lens, self.num_free = plan.seq_lens, plan.num_free
        return plan

    def go_on(self, parents: torch.Tensor, num_blocks: int, caches) -> None:
        """The batch becomes the rows `parents` of it (-1: none), each with a cache of its own to
        append to."""
        r = kv8.reorder(parents, self.lens, self.tables, self.free, self.num_free, self.block_size,
                        num_blocks)
        kv8.copy_blocks(caches, r.sources, r.targets)
        self.tables, self.lens, self.free, self.num_free = r[:4]


class Decoder:
    """Pre-norm decoder, rotary positions, grouped heads; every product is a packed linear."""

    def __init__(self, layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, vocabulary=1000,
                 dtype=torch.bfloat16, device="cuda", seed=0):
        gen = torch.Generator().manual_seed(seed)

        def linear(n_in, n_out, **kw):
            m = torch.nn.Linear(n_in, n_out, bias=False)
            with torch.no_grad():
                m.weight.copy_(torch.randn(n_out, n_in, generator=gen) * n_in ** -0.5)
            return E8LatticeLinear.from_linear(m.to(device=device, dtype=dtype), bitrate=2.0, **kw)

        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        self.embedding = torch.randn(vocabulary, hidden, generator=gen).to(device, dtype)
        self.qkv = [linear(hidden, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)]
        self.out = [linear(heads * head_dim, hidden) for _ in range(layers)]
        self.up = [linear(hidden, 4 * hidden) for _ in range(layers)]
        self.down = [linear(4 * hidden, hidden) for _ in range(layers)]
        self.head = linear(hidden, vocabulary, rank=8)
        self.rotation = rotary.rotation(head_dim, 10000.0, device=device)

    def caches(self, num_blocks, block_size):
        return [KV8Cache(num_blocks, self.kv_heads, self.head_dim, block_size,
                         self.embedding.device) for _ in self.qkv]

    def hidden(self, tokens, plan, tables, caches, rotate_on_append=False, **longest):
        """The tokens' last hidden states; their keys and values go into the caches, rotated before
        or on the way (then without a rounding between)."""
        x, t = self.embedding[tokens], len(tokens)
        q_size, kv_size = self.heads * self.head_dim, self.kv_heads * self.head_dim
        for i, cache in enumerate(caches):
            q, k, v = self.qkv[i](F.rms_norm(x, x.shape[-1:])).split([q_size, kv_size, kv_size], -1)
            q, k, v = (y.unflatten(-1, (-1, self.head_dim)) for y in (q, k, v))
            if rotate_on_append:
                q = cache.rotate_append(q, k, v, plan.positions, plan.slots, self.rotation)
            else:
                q, k = rotary.rotate_qk(q, k, plan.positions, self.rotation)
                cache.append(k, v, plan.slots)
            o = cache.attention(q, tables, plan.seq_lens, plan.query_starts, **longest)
            x = x + self.out[i](o.reshape(t, -1))
            x = x + self.down[i](F.silu(self.up[i](F.rms_norm(x, x.shape[-1:]))))
        return F.rms_norm(x, x.shape[-1:])


@torch.no_grad()
def answer(model: Decoder, prompts, new_tokens: int, num_blocks=64, block_size=16):
    """Greedy answers of ``new_tokens`` each.

    Returns (tokens [requests, new], their log probabilities, the prompts' log probabilities as
    one row of tokens, the hidden states the answers came from, the requests, the caches)."""
    device = model.embedding.device
    lens = [len(p) for p in prompts]
    batch = Requests(len(prompts), max(lens) + new_tokens, num_blocks, block_size, device)
    caches = model.caches(num_blocks, block_size)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    follow = torch.tensor([t for p in prompts for t in (*p[1:], -1)], device=device)  # -1: none
    plan = batch.step(torch.tensor(lens, dtype=torch.int32, device=device), len(tokens))
    h = model.hidden(tokens, plan, batch.tables, caches, max_query_len=max(lens),
                     max_seq_len=max(lens))
    prompt_logprobs = token_logprobs(model.head(h), follow).logprob

    states, chosen, logprobs = [h[plan.query_starts[1:].long() - 1]], [], []
    one = torch.ones(len(prompts), dtype=torch.int32, device=device)
    for i in range(new_tokens):
        logits = model.head(states[-1])
        # the most likely token; a sampler would pass its own choice as the ids
        best = token_logprobs(logits, torch.full_like(one, -1, dtype=torch.int64), top_k=1)
        chosen.append(best.top_ids[:, 0])
        logprobs.append(best.top_logprobs[:, 0])
        if i + 1 < new_tokens:
            plan = batch.step(one, len(prompts))
            states.append(model.hidden(chosen[-1], plan, batch.tables, caches, max_query_len=1,
                                       max_seq_len=max(lens) + i + 1))
    return (torch.stack(chosen, 1), torch.stack(logprobs, 1), prompt_logprobs,
            torch.stack(states, 1), batch, caches)


@torch.no_grad()
def beam_answer(model: Decoder, prompts, beams: int, new_tokens: int, end: int, num_blocks=256,
                block_size=16, watch=None):
    """The best answers of ``new_tokens`` tokens, less behind the token ``end``, by beam search.

    Returns (tokens [requests, beams, new], their log probabilities [requests, beams], the requests,
    the caches).  ``watch`` is called with each step's logits, scores, finished beams and choice."""
    device, n = model.embedding.device, len(prompts)
    lens = [len(p) for p in prompts]
    batch = Requests(n, max(lens) + new_tokens, num_blocks, block_size, device)
    caches = model.caches(num_blocks, block_size)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    plan = batch.step(torch.tensor(lens, dtype=torch.int32, device=device), len(tokens))
    h = model.hidden(tokens, plan, batch.tables, caches, True, max_query_len=max(lens),
                     max_seq_len=max(lens))[plan.query_starts[1:].long() - 1]
    scores = torch.zeros(n, 1, device=device)
    done = torch.zeros(n, 1, dtype=torch.bool, device=device)
    answers = torch.zeros(n, 0, dtype=torch.int64, device=device)
    one = torch.ones(n * beams, dtype=torch.int32, device=device)
    for i in range(new_tokens):
        logits = model.head(h).unflatten(0, scores.shape)
        best = beam_select(logits, scores, beams, finished=done, pad_id=end)
        if watch is not None:
            watch(logits, scores, done, best)
        rows, scores = best.parents.flatten(), best.scores
        done = done.flatten()[best.parents] | (best.tokens == end)
        answers = torch.cat([answers[rows], best.tokens.flatten()[:, None]], 1)
        batch.go_on(rows, num_blocks, caches)
        if i + 1 < new_tokens:
            plan = batch.step(one, n * beams)
            h = model.hidden(answers[:, -1], plan, batch.tables, caches, True, max_query_len=1,
                             max_seq_len=max(lens) + i + 1)
    return answers.unflatten(0, (n, beams)), scores, batch, caches


def reinforce(model: Decoder, states, tokens, old_logprobs, rewards, steps=4, rate=1e-2,
              entropy_weight=1e-3):
    """Policy steps on the head's adapter: a clipped ratio of each token's probability now to
    then, with the entropy's bonus.  Returns each step's loss."""
    params = [p for p in (model.head.lora_A, model.head.lora_B) if p is not None]
    optimizer = torch.optim.SGD(params, lr=rate)
    gain = (rewards - rewards.mean())[:, None]
    losses = []
    for _ in range(steps):
        now = token_logprobs(model.head(states), tokens)
        ratio = (now.logprob - old_logprobs).exp()
        loss = -torch.minimum(ratio * gain, ratio.clamp(0.8, 1.2) * gain).mean()
        loss = loss - entropy_weight * now.entropy.mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses)


def main() -> None:
    model = Decoder()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (1, 37, 16, 120)]
    tokens, logprobs, prompt_logprobs, states, batch, _ = answer(model, prompts, 24)
    print("answers", tokens[:, :8].tolist())
    print("their log probabilities", [round(v, 3) for v in logprobs.sum(1).tolist()])
    print("prompts' log probability", round(prompt_logprobs.sum().item(), 3))
    print("blocks left", batch.num_free.item())
    rewards = (tokens % 2 == 0).float().mean(1)
    print("losses", [round(v, 5) for v in reinforce(model, states, tokens, logprobs,
                                                    rewards).tolist()])
    answers, scores, batch, caches = beam_answer(model, prompts, 4, 12, end=7)
    print("best of four beams", answers[:, 0, :8].tolist())
    print("their log probabilities", [round(v, 3) for v in scores[:, 0].tolist()])
    batch.go_on(torch.full((16,), -1, device=tokens.device), 256, caches)
    print("blocks given back", batch.num_free.item())


if __name__ == "__main__":
    main()
