"""An 8-bit paged key / value cache for decoders of packed linears, and attention over it.

Keys and values are held as int8 codes with one float32 scale for each block of tokens and head
(``include/ojasx_e8t.h`` has the layout).  One step of a batch:

    p = kv8.plan(seq_lens, new_lens, block_tables, free_blocks, num_free, block_size, num_tokens)
    cache.append(k, v, p.slots)                      # for each layer; or, with positions rotated
    q = cache.rotate_append(q, k, v, p.positions, p.slots, rotation)    # in on the way
    o = cache.attention(q, block_tables, p.seq_lens, p.query_starts)

``plan`` runs on the GPU from the requests' lengths alone, so a step needs no copy to the host;
``KV8Cache`` is one layer's storage.  The functions take the storage's tensors, for callers that keep
them in tensors of their own.  Requests that go on from others (beams, several answers to one
prompt) or are done share and give back blocks:

    r = kv8.reorder(parents, seq_lens, block_tables, free_blocks, num_free, block_size, num_blocks)
    kv8.copy_blocks(caches, r.sources, r.targets)    # what begun blocks hold, in all layers
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from . import serve_ops as S
from .rotary import Rotation


def _eager(name: str, *args):
    """The call in native code where it is plain eager work, else None (csrc/e8t_torch.cpp)."""
    return None if torch.compiler.is_compiling() else getattr(N.eager(), name)(*args)


class KV8Plan(NamedTuple):
    """Where a step's tokens go (``plan``).

    The results may share allocations: one for up to 64 KiB of them, else one for the three of each
    token and one for the others.  ``clone()`` what is to be resized in place, or kept alone."""

    slots: torch.Tensor         # int64 [tokens]: block * block_size + offset, -1 without a block
    positions: torch.Tensor     # int32 [tokens]: place in the request
    requests: torch.Tensor      # int32 [tokens]
    query_starts: torch.Tensor  # int32 [requests + 1]: first token of each request
    seq_lens: torch.Tensor      # int32 [requests]: lengths after the step
    num_free: torch.Tensor      # int32 [1]: blocks left; negative: so many were missing


def plan(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
         free_blocks: torch.Tensor, num_free: torch.Tensor, block_size: int,
         num_tokens: int) -> KV8Plan:
    """Blocks and slots for ``new_lens`` more tokens of requests that hold ``seq_lens``.

    Blocks that the new tokens begin come from the top of the stack ``free_blocks[:num_free]`` and
    are entered in ``block_tables`` (int32 ``[requests, blocks]``, in place).  The stack itself is
    not written: pass the returned ``num_free`` to the next call.  ``num_tokens`` is the sum of
    ``new_lens`` or more (a padded batch); of more new tokens only the first ``num_tokens`` get
    their place.
    """
    args = (seq_lens, new_lens, block_tables, free_blocks, num_free, block_size, num_tokens)
    return KV8Plan(*(_eager("kv8_plan", *args) or S.kv8_plan(*args)))


class KV8Reorder(NamedTuple):
    """A batch after ``reorder``.  The results may share allocations (see ``KV8Plan``)."""

    block_tables: torch.Tensor  # int32 [new rows, blocks], -1 behind a row's blocks
    seq_lens: torch.Tensor      # int32 [new rows]
    free_blocks: torch.Tensor   # int32 [num_blocks], -1 from num_free on
    num_free: torch.Tensor      # int32 [1]; negative: so many blocks were missing
    sources: torch.Tensor       # int32 [new rows]: begun blocks to be copied, -1 for none
    targets: torch.Tensor       # int32 [new rows]: where to


def reorder(parents: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
            free_blocks: torch.Tensor, num_free: torch.Tensor, block_size: int, num_blocks: int
            ) -> KV8Reorder:
    """The batch whose row i goes on from row ``parents[i]`` (int64; -1: an empty row) of this one.

    There may be more or fewer rows than before (up to 2^25): ``[0, 0, 0, 0]`` makes four beams of a
    prompt.  Children of a row share its full blocks.  Its begun block stays with the first of them,
    the others get one each from the stack: ``copy_blocks`` copies what it holds, in all layers, before
    the next append.  Blocks that no new row holds go back on the stack, before any is taken.

    All rows that share a block have to be in one call, since blocks are freed by what its rows
    hold; a begun block is held by one row alone, as this and ``plan`` leave it.  Nothing is written
    in place.  The stack returned has room for all ``num_blocks``.
    """
    args = (parents, seq_lens, block_tables, free_blocks, num_free, block_size, num_blocks)
    return KV8Reorder(*(_eager("kv8_reorder", *args) or S.kv8_reorder(*args)))


def copy_blocks(caches: Sequence, sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Copies blocks ``sources[i]`` to ``targets[i]`` in every one of ``caches``: ``KV8Cache`` objects,
    or triples of their tensors, all of one shape.  Pairs with a block outside the cache (-1) are
    skipped.  No block may be a target twice, or a target and a source."""
    if _eager("kv8_copy_blocks", caches, sources, targets) is not None:
        return
    parts = [(c.k_codes, c.v_codes, c.scales) if isinstance(c, KV8Cache) else tuple(c) for c in caches]
    if any(len(p) != 3 for p in parts):
        raise RuntimeError("a cache is a KV8Cache or its three tensors")
    S.kv8_copy_blocks(*([p[i] for p in parts] for i in range(3)), sources, targets)


def append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_codes: torch.Tensor,
           v_codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Writes ``k``, ``v`` ``[tokens, kv heads, head size]`` into the cache at ``slots``.

    A block's scale covers the largest element it was given; where a later token raises it, the
    codes that are there already are rounded again.  Slots outside the cache (-1) are skipped.

    In one call the tokens of a block have to be neighbours in ``slots``, at rising offsets without
    a gap, as ``plan`` gives them: one run for each block.  Two runs of a block (slots 5, -1, 6 of
    one; a slot given twice) are written by different waves at once, and which scale and codes stay
    is undefined.  Append them in two calls.
    """
    args = (k, v, slots, k_codes, v_codes, scales)
    if _eager("kv8_append", *args) is None:
        S.kv8_append(*args)


def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  slots: torch.Tensor, rotation: Rotation, k_codes: torch.Tensor,
                  v_codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``append`` with ``positions`` ``[tokens]`` (int32 or int64) rotated into the keys on the way;
    returns ``q [tokens, heads, head size]`` rotated alike (``rotary.rotate`` has the rule).

    Rotated keys are not rounded to their type before they become codes: the cache then holds what
    ``append`` makes of keys that were rotated in float32.  No gradient passes.
    """
    args = (q, k, v, positions, slots, rotation.rates, rotation.gain, rotation.interleaved, k_codes,
            v_codes, scales)
    out = _eager("kv8_rotate_append", *args)
    return S.kv8_rotate_append(*args) if out is None else out


def read(k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor, blocks: torch.Tensor,
         head_dim: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keys and values of whole blocks, ``[n, block_size, kv heads, head size]`` in ``dtype``, and
    the blocks' scales ``[n, kv heads, 2]``."""
    args = (k_codes, v_codes, scales, blocks, head_dim)
    out = _eager("kv8_read", *args, N.DTYPE_CODE.get(dtype, -1))
    return S.kv8_read(*args, dtype) if out is None else out


def attention(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor,
              block_tables: torch.Tensor, seq_lens: torch.Tensor,
              query_starts: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
              window: int = 0, max_query_len: Optional[int] = None,
              max_seq_len: Optional[int] = None, return_lse: bool = False
              ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of the newest tokens ``q [tokens, heads, head size]`` over the cache.

    Request r's rows of ``q`` are ``query_starts[r]:query_starts[r + 1]`` (one each without
    ``query_starts``), its last tokens; ``seq_lens`` counts them too.  ``window``: only so many
    keys up to the token itself (0: all).  ``scale`` defaults to head size ** -0.5.
    ``max_query_len`` and ``max_seq_len`` are the batch's longest, where the caller knows them:
    they size the launch, and longer ones are cut off: of a request's rows the first
    ``max_query_len`` are computed, over its first ``max_seq_len`` keys.  A row that sees nothing is
    zero (log-sum -inf), and so are rows beyond ``max_query_len`` and tokens of no request (a padded
    batch).  With ``return_lse`` also the natural log of each row's softmax sum.

    Sums are in 32 bits.  float32 queries keep their 24 bits throughout; 16-bit ones enter the
    products as 16-bit fixed point of their row's largest element (rounded by 2^-16 of it at most).
    Their weights are rounded to 16 bits of the largest of 64 keys for few rows of a request, to
    fp16 for many (2^-11 each, denormal under 2^-14 of the row's reference).
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if max_query_len is None:
        max_query_len = 1 if query_starts is None else q.shape[0]
    if max_seq_len is None:
        max_seq_len = block_tables.shape[-1] * k_codes.shape[2]
    args = (q, k_codes, v_codes, scales, block_tables, seq_lens, query_starts, float(scale), window,
            max_query_len, max_seq_len, return_lse)
    out, lse = _eager("kv8_attention", *args) or S.kv8_attention(*args)
    return (out, lse) if return_lse else out


class KV8Cache:
    """One layer's storage: ``num_blocks`` blocks of ``block_size`` tokens (16, 32, 64, 128 or
    256) for ``kv_heads`` heads of ``head_dim`` (1..256)."""

    def __init__(self, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64,
                 device: Union[str, torch.device, None] = "cuda"):
        S._check_block_size(block_size)
        if not 1 <= head_dim <= S.MAX_HEAD_DIM or num_blocks < 0 or kv_heads < 1:
            raise RuntimeError(f"no cache of {num_blocks} blocks for {kv_heads} heads of {head_dim}")
        shape = (num_blocks, kv_heads, block_size, S.stored_dim(head_dim))
        self.head_dim, self.block_size = head_dim, block_size
        self.k_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.v_codes = torch.zeros(shape, dtype=torch.int8, device=device)
        self.scales = torch.zeros((num_blocks, kv_heads, 2), dtype=torch.float32, device=device)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """``kv8.append`` into this storage: the tokens of a block in one run of ``slots``."""
        append(k, v, slots, self.k_codes, self.v_codes, self.scales)

    def rotate_append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, rotation: Rotation
                      ) -> torch.Tensor:
        """``kv8.rotate_append`` into this storage; returns the rotated queries."""
        return rotate_append(q, k, v, positions, slots, rotation, self.k_codes, self.v_codes,
                             self.scales)

    def read(self, blocks: torch.Tensor, dtype: torch.dtype = torch.bfloat16
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        return read(self.k_codes, self.v_codes, self.scales, blocks, self.head_dim, dtype)

    def attention(self, q: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  query_starts: Optional[torch.Tensor] = None, **kwargs):
        return attention(q, self.k_codes, self.v_codes, self.scales, block_tables, seq_lens,
                         query_starts, **kwargs)
