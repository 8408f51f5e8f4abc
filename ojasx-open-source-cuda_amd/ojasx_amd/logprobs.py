"""Log probabilities of given tokens, with entropy and the most likely alternatives."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from . import serve_ops as S


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``.

    They may share allocations: one for up to 64 KiB of them, else one for those of each row and one
    for the alternatives.  ``clone()`` what is to be resized in place, or kept alone."""

    logprob: torch.Tensor       # float32 [...]: of the given tokens
    entropy: torch.Tensor       # float32 [...]: of the rows' distributions, in nats
    lse: torch.Tensor           # float32 [...]: log of the sum of exp(logits)
    top_logprobs: torch.Tensor  # float32 [..., top_k], falling
    top_ids: torch.Tensor       # int64 [..., top_k]; equal logits by rising token


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Of ``logits [..., vocabulary]`` and tokens ``ids [...]`` (int64), in one pass.

    An id outside the vocabulary (-100, -1) has log probability 0 and no gradient.  Masked logits
    (-inf) have probability 0; a row of nothing else gives lse -inf, entropy 0.  ``top_k`` up to
    64.  All float results pass their gradients to ``logits`` (once: the gradient itself cannot be
    differentiated); sums are in float32 whatever the logits' type.
    """
    if not torch.compiler.is_compiling():
        e = N.eager()  # None: with a gradient to record; not plain eager work at all
        out = e.token_logprobs(logits, ids, top_k) or e.token_logprobs_recorded(logits, ids, top_k)
        if out is not None:
            return TokenLogprobs(*out[:5])
    return TokenLogprobs(*S.token_logprobs(logits, ids, top_k)[:5])
