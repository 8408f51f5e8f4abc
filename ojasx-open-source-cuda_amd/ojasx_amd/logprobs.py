"""Log probabilities of given tokens, with entropy and the most likely alternatives."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from . import serve_ops as S


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # float32 [...]: of the given tokens
    entropy: torch.Tensor       # float32 [...]: of the rows' distributions, in nats
    lse: torch.Tensor           # float32 [...]: log of the sum of exp(logits)
    top_logprobs: torch.Tensor  # float32 [..., top_k], falling
    top_ids: torch.Tensor       # int64 [..., top_k]; equal logits by rising token


class _Recorded(torch.autograd.Function):
    """token_logprobs recorded for plain eager calls (the registered op's own autograd formula,
    without the ops' dispatch)."""

    @staticmethod
    def forward(ctx, logits, ids, top_k):
        out = N.eager().token_logprobs(logits, ids, top_k)
        if out is None:
            out = S.token_logprobs(logits, ids, top_k)
        lp, entropy, lse, top, top_ids, stats = out
        ctx.save_for_backward(logits, ids, entropy, stats, top_ids)
        ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return lp, entropy, lse, top, top_ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        grads = grads[:4]
        if all(g is None for g in grads):
            return None, None, None
        args = (*ctx.saved_tensors, *grads)
        gx = N.eager().token_logprobs_bwd(*args)
        return S.token_logprobs_bwd(*args) if gx is None else gx, None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Of ``logits [..., vocabulary]`` and tokens ``ids [...]`` (int64), in one pass.

    An id outside the vocabulary (-100, -1) has log probability 0 and no gradient.  Masked logits
    (-inf) have probability 0; a row of nothing else gives lse -inf, entropy 0.  ``top_k`` up to
    64.  All float results pass their gradients to ``logits`` (once: the gradient itself cannot be
    differentiated); sums are in float32 whatever the logits' type.
    """
    if not torch.compiler.is_compiling():
        out = N.eager().token_logprobs(logits, ids, top_k)  # None: to be recorded, or not plain
        if out is not None:
            return TokenLogprobs(*out[:5])
        if N.eager().is_plain(logits, ids):
            return TokenLogprobs(*_Recorded.apply(logits, ids, top_k))
    return TokenLogprobs(*S.token_logprobs(logits, ids, top_k)[:5])
