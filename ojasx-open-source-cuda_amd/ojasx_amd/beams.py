"""Beam search: the best continuations of each group of beams over its beams and the vocabulary.

    step = beam_select(logits, scores, num=beams, finished=done, pad_id=0)
    state = state[step.parents.flatten()]          # what each beam carries along
    r = kv8.reorder(step.parents.flatten(), ...)   # its cache: blocks are shared, not copied
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N
from . import serve_ops as S


class BeamStep(NamedTuple):
    """Results of ``beam_select``.  They may share an allocation: ``clone()`` what is kept alone."""

    scores: torch.Tensor   # float32 [groups, num], falling
    parents: torch.Tensor  # int64 [groups, num]: row (group * beams + beam) that is continued
    tokens: torch.Tensor   # int64 [groups, num]


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None, pad_id: int = 0) -> BeamStep:
    """The ``num`` (default: as many as beams; up to 64) best continuations of each group.

    ``logits [groups, beams, vocabulary]`` (up to 64 beams, fewer than 2^23 in all groups), ``scores``
    float32 ``[groups, beams]``: the beams' log probabilities so far.  A continuation's value is its
    beam's score plus the token's log probability; equal ones come by rising beam, of one beam by
    falling logit (beside a score like -1e30 all of a beam's values are one), then by rising token.  A
    beam that is ``finished`` (bool ``[groups, beams]``) goes on by ``pad_id`` alone, at its score, and
    its logits are not read.

    A group's first step, with all beams alike, is chosen from one: scores of -inf for the others.
    Impossible continuations (masked logits of -inf, such scores) are taken, in the order of beams
    and tokens at a score of -inf, where a group has fewer than ``num`` others.  A beam with a score
    or a logit of NaN or +inf has NaN continuations, which come first, by rising token.

    Values are compared in 64 bits, so the choice does not hang on the rounding of 32-bit sums (they
    are formed again in 64 where two beams' values are closer than 2^-18, or than 2^-50 of
    themselves); they are returned rounded to float32.  No gradient passes.
    """
    if num is None:
        num = logits.shape[1] if logits.dim() == 3 else 1  # (others are refused)
    if not torch.compiler.is_compiling():
        out = N.eager().beam_select(logits, scores, num, finished, pad_id)
        if out is not None:
            return BeamStep(*out)
    return BeamStep(*S.beam_select(logits, scores, num, finished, pad_id))
