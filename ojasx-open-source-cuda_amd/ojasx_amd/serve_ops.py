"""``torch.library`` custom ops (namespace ``ojasx_e8t``) of the operators around the packed
linears: the 8-bit paged key / value cache, its attention, token log probabilities, rotated
positions, beam search.

``kv8_plan``, ``kv8_append`` (a block's tokens in one run of its slots) and ``kv8_read`` move a
step's tokens into the cache and blocks out of it (``kv8_rotate_append`` with positions rotated into
keys and queries on the way), ``kv8_reorder`` and ``kv8_copy_blocks`` let requests go on from
others, ``kv8_attention`` reads it; ``rotary`` (its own gradient, turned back) rotates queries and
keys; ``beam_select`` chooses the beams that go on; ``token_logprobs`` (autograd registered, with
``token_logprobs_bwd``) is what a model answers and trains with.  The reference keeps no quantized
cache; the layouts and rules are those of ``include/ojasx_e8t.h``.  As for the other ops: the current
HIP stream of the device, outputs and workspaces from torch's caching allocator, ``RuntimeError`` for
what does not fit, no fallback.
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch

from . import _native as N
from .ops import _NS, _dtype_code

BLOCK_SIZES = (16, 32, 64, 128, 256)
MAX_HEAD_DIM = 256
MAX_TOP = 64
MAX_BEAMS = 64


def stored_dim(head_dim: int) -> int:
    """Bytes that the cache keeps of a head: its size rounded up to a multiple of 64."""
    return (head_dim + 63) // 64 * 64


def _ints(what: str, t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, ...]) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise RuntimeError(f"{what} must be {dtype} of shape {list(shape)} "
                           f"(got {t.dtype} {list(t.shape)})")
    return t.contiguous()


def _check_block_size(block_size: int) -> None:
    if block_size not in BLOCK_SIZES:
        raise RuntimeError(f"block_size must be one of {BLOCK_SIZES} (got {block_size})")


def _check_cache(k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor,
                 head_dim: int) -> Tuple[int, int, int]:
    """(blocks, kv heads, block size) of a cache; its tensors are taken as they lie."""
    if k_codes.dtype != torch.int8 or v_codes.dtype != torch.int8 or scales.dtype != torch.float32:
        raise RuntimeError("a cache is int8 codes with float32 scales")
    if k_codes.dim() != 4 or v_codes.shape != k_codes.shape:
        raise RuntimeError("k_codes and v_codes must be [blocks, kv heads, block size, stored dim] "
                           f"(got {list(k_codes.shape)} and {list(v_codes.shape)})")
    blocks, heads, block_size, dp = k_codes.shape
    if tuple(scales.shape) != (blocks, heads, 2):
        raise RuntimeError(f"scales must be {[blocks, heads, 2]} (got {list(scales.shape)})")
    if not (k_codes.is_contiguous() and v_codes.is_contiguous() and scales.is_contiguous()):
        raise RuntimeError("a cache's tensors must be contiguous")
    _check_block_size(block_size)
    if not 1 <= head_dim <= MAX_HEAD_DIM or dp != stored_dim(head_dim):
        raise RuntimeError(f"head size {head_dim} does not fit a cache that stores {dp} "
                           f"(1..{MAX_HEAD_DIM}, rounded up to a multiple of 64)")
    return blocks, heads, block_size


def _table(block_tables: torch.Tensor, requests: int) -> torch.Tensor:
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or \
            block_tables.shape[0] != requests:
        raise RuntimeError(f"block_tables must be int32 [{requests}, blocks] "
                           f"(got {block_tables.dtype} {list(block_tables.shape)})")
    return block_tables


# ----------------------------------------------------------------------------- plan

@torch.library.custom_op(f"{_NS}::kv8_plan", mutates_args=("block_tables",))
def kv8_plan(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
             free_blocks: torch.Tensor, num_free: torch.Tensor, block_size: int, num_tokens: int
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                        torch.Tensor]:
    dev = N.require_device(seq_lens, new_lens, block_tables, free_blocks, num_free)
    r = seq_lens.numel()
    seq = _ints("seq_lens", seq_lens, torch.int32, (r,))
    new = _ints("new_lens", new_lens, torch.int32, (r,))
    free = _ints("free_blocks", free_blocks, torch.int32, (free_blocks.numel(),))
    nf = _ints("num_free", num_free, torch.int32, (1,))
    _table(block_tables, r)
    if block_tables.numel() and block_tables.stride(1) != 1:
        raise RuntimeError("block_tables is written in place: its columns must be neighbours")
    _check_block_size(block_size)
    if num_tokens < 0:
        raise RuntimeError(f"num_tokens is {num_tokens}")
    i32 = dict(dtype=torch.int32, device=dev)
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    positions, requests = torch.empty(num_tokens, **i32), torch.empty(num_tokens, **i32)
    starts, lens, left = torch.empty(r + 1, **i32), torch.empty(r, **i32), torch.empty(1, **i32)
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_kv8_plan(
            N.ptr(seq), N.ptr(new), r, N.ptr(block_tables), block_tables.stride(0),
            block_tables.shape[1], N.ptr(free), free.numel(), N.ptr(nf), block_size, num_tokens,
            N.ptr(slots), N.ptr(positions), N.ptr(requests), N.ptr(starts), N.ptr(lens),
            N.ptr(left), N.stream_handle(dev)), "kv8_plan")
    return slots, positions, requests, starts, lens, left


@kv8_plan.register_fake
def _(seq_lens, new_lens, block_tables, free_blocks, num_free, block_size, num_tokens):
    r = seq_lens.numel()
    return (seq_lens.new_empty(num_tokens, dtype=torch.int64), seq_lens.new_empty(num_tokens),
            seq_lens.new_empty(num_tokens), seq_lens.new_empty(r + 1), seq_lens.new_empty(r),
            seq_lens.new_empty(1))


# ----------------------------------------------------------------------------- append, read

def _rows(what: str, t: torch.Tensor, tokens: int, heads: int) -> torch.Tensor:
    """[tokens, heads, d] with neighbouring d, as it lies where it can be."""
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[1] != heads:
        raise RuntimeError(f"{what} must be [{tokens}, {heads}, head size] (got {list(t.shape)})")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


@torch.library.custom_op(f"{_NS}::kv8_append", mutates_args=("k_codes", "v_codes", "scales"))
def kv8_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_codes: torch.Tensor,
               v_codes: torch.Tensor, scales: torch.Tensor) -> None:
    dev = N.require_device(k, v, slots, k_codes, v_codes, scales)
    dt = _dtype_code(k.dtype)
    if v.dtype != k.dtype or k.dim() != 3 or v.shape != k.shape:
        raise RuntimeError(f"k and v must be [tokens, kv heads, head size] of one type "
                           f"(got {k.dtype} {list(k.shape)} and {v.dtype} {list(v.shape)})")
    t, _, d = k.shape
    blocks, heads, block_size = _check_cache(k_codes, v_codes, scales, d)
    kr, vr = _rows("k", k, t, heads), _rows("v", v, t, heads)
    s = _ints("slots", slots, torch.int64, (t,))
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_kv8_append(
            N.ptr(k_codes), N.ptr(v_codes), N.ptr(scales), blocks, heads, block_size, d,
            N.ptr(kr), kr.stride(0), kr.stride(1), N.ptr(vr), vr.stride(0), vr.stride(1), dt,
            N.ptr(s), t, N.stream_handle(dev)), "kv8_append")


@kv8_append.register_fake
def _(k, v, slots, k_codes, v_codes, scales):
    return None


@torch.library.custom_op(f"{_NS}::kv8_read", mutates_args=())
def kv8_read(k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor,
             blocks: torch.Tensor, head_dim: int, dtype: torch.dtype
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dev = N.require_device(k_codes, v_codes, scales, blocks)
    dt = _dtype_code(dtype)
    num_blocks, heads, block_size = _check_cache(k_codes, v_codes, scales, head_dim)
    b = _ints("blocks", blocks, torch.int32, (blocks.numel(),))
    k = torch.empty((b.numel(), block_size, heads, head_dim), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    s = torch.empty((b.numel(), heads, 2), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_kv8_read(
            N.ptr(k_codes), N.ptr(v_codes), N.ptr(scales), num_blocks, heads, block_size, head_dim,
            N.ptr(b), b.numel(), dt, N.ptr(k), N.ptr(v), N.ptr(s), N.stream_handle(dev)), "kv8_read")
    return k, v, s


@kv8_read.register_fake
def _(k_codes, v_codes, scales, blocks, head_dim, dtype):
    shape = (blocks.numel(), k_codes.shape[2], k_codes.shape[1], head_dim)
    return (k_codes.new_empty(shape, dtype=dtype), k_codes.new_empty(shape, dtype=dtype),
            scales.new_empty((blocks.numel(), k_codes.shape[1], 2)))


@torch.library.custom_op(f"{_NS}::kv8_rotate_append",
                         mutates_args=("k_codes", "v_codes", "scales"))
def kv8_rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                      slots: torch.Tensor, rates: torch.Tensor, gain: float, interleaved: bool,
                      k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor
                      ) -> torch.Tensor:
    dev = N.require_device(q, k, v, positions, slots, rates, k_codes, v_codes, scales)
    dt = _dtype_code(k.dtype)
    if v.dtype != k.dtype or k.dim() != 3 or v.shape != k.shape:
        raise RuntimeError(f"k and v must be [tokens, kv heads, head size] of one type "
                           f"(got {k.dtype} {list(k.shape)} and {v.dtype} {list(v.shape)})")
    t, _, d = k.shape
    if q.dtype != k.dtype or q.dim() != 3 or q.shape[0] != t or q.shape[2] != d:
        raise RuntimeError(f"q must be {k.dtype} {[t, 'heads', d]} (got {q.dtype} {list(q.shape)})")
    blocks, heads, block_size = _check_cache(k_codes, v_codes, scales, d)
    kr, vr = _rows("k", k, t, heads), _rows("v", v, t, heads)
    s = _ints("slots", slots, torch.int64, (t,))
    if positions.dim() != 1:
        raise RuntimeError(f"positions must be [{t}] (got {list(positions.shape)})")
    _check_rotation(positions, (t,), rates, d)
    qr, p = _rotary_input(q), positions.contiguous()
    out = _rotary_output(qr)
    rot = N.Rotation(N.ptr(rates), rates.numel(), N.ptr(p), p.dtype == torch.int64, interleaved,
                     gain, False)
    rows = _rotary_rows(qr, out)
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_kv8_rotate_append(
            N.ptr(k_codes), N.ptr(v_codes), N.ptr(scales), blocks, heads, block_size, d,
            N.ptr(kr), kr.stride(0), kr.stride(1), N.ptr(vr), vr.stride(0), vr.stride(1), dt,
            N.ptr(s), t, ctypes.byref(rows), ctypes.byref(rot), N.stream_handle(dev)),
            "kv8_rotate_append")
    return out


@kv8_rotate_append.register_fake
def _(q, k, v, positions, slots, rates, gain, interleaved, k_codes, v_codes, scales):
    return _rotary_output(_rotary_input(q))


# ----------------------------------------------------------------------------- reorder

@torch.library.custom_op(f"{_NS}::kv8_reorder", mutates_args=())
def kv8_reorder(parents: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
                free_blocks: torch.Tensor, num_free: torch.Tensor, block_size: int, num_blocks: int
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                           torch.Tensor]:
    """(tables, lengths, stack, its size, sources, targets) of the rows that continue `parents`."""
    dev = N.require_device(parents, seq_lens, block_tables, free_blocks, num_free)
    r, c = seq_lens.numel(), parents.numel()
    par = _ints("parents", parents, torch.int64, (c,))
    seq = _ints("seq_lens", seq_lens, torch.int32, (r,))
    free = _ints("free_blocks", free_blocks, torch.int32, (free_blocks.numel(),))
    nf = _ints("num_free", num_free, torch.int32, (1,))
    tables = _table(block_tables, r)
    if tables.numel() and tables.stride(1) != 1:
        tables = tables.contiguous()
    _check_block_size(block_size)
    if num_blocks < 0:
        raise RuntimeError(f"num_blocks is {num_blocks}")
    i32 = dict(dtype=torch.int32, device=dev)
    w = tables.shape[1]
    out = (torch.empty((c, w), **i32), torch.empty(c, **i32), torch.empty(num_blocks, **i32),
           torch.empty(1, **i32), torch.empty(c, **i32), torch.empty(c, **i32))
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        N.check(N.lib().ojx_kv8_reorder_workspace_bytes(r, c, w, block_size, num_blocks,
                                                        ctypes.byref(nbytes)),
                "kv8_reorder_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        N.check(N.lib().ojx_kv8_reorder(
            N.ptr(par), c, N.ptr(seq), r, N.ptr(tables), tables.stride(0), w, N.ptr(free),
            free.numel(), N.ptr(nf), block_size, num_blocks, *(N.ptr(t) for t in out), N.ptr(ws),
            nbytes.value, N.stream_handle(dev)), "kv8_reorder")
    return out


@kv8_reorder.register_fake
def _(parents, seq_lens, block_tables, free_blocks, num_free, block_size, num_blocks):
    c = parents.numel()
    return (block_tables.new_empty((c, block_tables.shape[1])), seq_lens.new_empty(c),
            seq_lens.new_empty(num_blocks), seq_lens.new_empty(1), seq_lens.new_empty(c),
            seq_lens.new_empty(c))


@torch.library.custom_op(f"{_NS}::kv8_copy_blocks", mutates_args=("k_codes", "v_codes", "scales"))
def kv8_copy_blocks(k_codes: List[torch.Tensor], v_codes: List[torch.Tensor],
                    scales: List[torch.Tensor], sources: torch.Tensor, targets: torch.Tensor
                    ) -> None:
    dev = N.require_device(*k_codes, *v_codes, *scales, sources, targets)
    n = sources.numel()
    src, dst = _ints("sources", sources, torch.int32, (n,)), _ints("targets", targets, torch.int32, (n,))
    if not len(k_codes) == len(v_codes) == len(scales):
        raise RuntimeError(f"{len(k_codes)}, {len(v_codes)} and {len(scales)} tensors of caches")
    if not k_codes:
        return
    for k, v, s in zip(k_codes, v_codes, scales):
        if k.shape != k_codes[0].shape:
            raise RuntimeError(f"caches of one call must be of one shape (got {list(k.shape)} and "
                               f"{list(k_codes[0].shape)})")
        blocks, heads, block_size = _check_cache(k, v, s, k.shape[-1])
    caches = (N.KV8Storage * len(k_codes))(*((N.ptr(k), N.ptr(v), N.ptr(s))
                                             for k, v, s in zip(k_codes, v_codes, scales)))
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_kv8_copy_blocks(
            caches, len(k_codes), blocks, heads, block_size, k_codes[0].shape[-1], N.ptr(src),
            N.ptr(dst), n, N.stream_handle(dev)), "kv8_copy_blocks")


@kv8_copy_blocks.register_fake
def _(k_codes, v_codes, scales, sources, targets):
    return None


# ----------------------------------------------------------------------------- attention

@torch.library.custom_op(f"{_NS}::kv8_attention", mutates_args=())
def kv8_attention(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                  scales: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  query_starts: Optional[torch.Tensor], scale: float, window: int,
                  max_query_len: int, max_seq_len: int, return_lse: bool
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    dev = N.require_device(q, k_codes, v_codes, scales, block_tables, seq_lens, query_starts)
    dt = _dtype_code(q.dtype)
    if q.dim() != 3:
        raise RuntimeError(f"q must be [tokens, heads, head size] (got {list(q.shape)})")
    t, heads, d = q.shape
    blocks, kv_heads, block_size = _check_cache(k_codes, v_codes, scales, d)
    qr = _rows("q", q, t, heads)
    r = seq_lens.numel()
    lens = _ints("seq_lens", seq_lens, torch.int32, (r,))
    starts = None
    if query_starts is not None:
        starts = _ints("query_starts", query_starts, torch.int32, (r + 1,))
    tables = _table(block_tables, r)
    if tables.numel() and tables.stride(1) != 1:
        tables = tables.contiguous()
    out = torch.empty((t, heads, d), dtype=q.dtype, device=dev)
    lse = torch.empty((t, heads) if return_lse else (0, heads), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        N.check(N.lib().ojx_kv8_attention_workspace_bytes(
            t, r, heads, kv_heads, d, window, max_query_len, max_seq_len, dt,
            ctypes.byref(nbytes)), "kv8_attention_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        N.check(N.lib().ojx_kv8_attention(
            N.ptr(qr), qr.stride(0), qr.stride(1), t, heads, dt, N.ptr(k_codes), N.ptr(v_codes),
            N.ptr(scales), blocks, kv_heads, block_size, d, N.ptr(tables), tables.stride(0),
            tables.shape[1], N.ptr(lens), N.ptr(starts), r, max_query_len, max_seq_len, scale,
            window, N.ptr(out), N.ptr(lse) if return_lse else 0, N.ptr(ws), nbytes.value,
            N.stream_handle(dev)), "kv8_attention")
    return out, lse


@kv8_attention.register_fake
def _(q, k_codes, v_codes, scales, block_tables, seq_lens, query_starts, scale, window,
      max_query_len, max_seq_len, return_lse):
    t, heads, _ = q.shape
    return (q.new_empty(q.shape), q.new_empty((t, heads) if return_lse else (0, heads),
                                              dtype=torch.float32))


# ----------------------------------------------------------------------------- log probabilities

def _logit_rows(logits: torch.Tensor, ids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"logits are {list(logits.shape)}, expected [..., vocabulary]")
    if ids.shape != logits.shape[:-1] or ids.dtype != torch.int64:
        raise RuntimeError(f"ids must be int64 {list(logits.shape[:-1])} "
                           f"(got {ids.dtype} {list(ids.shape)})")
    x = logits.reshape(-1, logits.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x, ids.reshape(-1).contiguous()


@torch.library.custom_op(f"{_NS}::token_logprobs", mutates_args=())
def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                              torch.Tensor, torch.Tensor]:
    """(logprob, entropy, lse, top_logprobs, top_ids, stats) of logits [..., V] and ids [...];
    stats [..., 2] is what the backward needs of the sum."""
    dev = N.require_device(logits, ids)
    dt = _dtype_code(logits.dtype)
    x, tokens = _logit_rows(logits, ids)
    rows, v = x.shape
    if not 0 <= top_k <= min(MAX_TOP, v):
        raise RuntimeError(f"top_k is {top_k}, expected 0..{min(MAX_TOP, v)}")
    f32 = dict(dtype=torch.float32, device=dev)
    lp, h, lse = torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty(rows, **f32)
    stats, top = torch.empty((rows, 2), **f32), torch.empty((rows, top_k), **f32)
    top_ids = torch.empty((rows, top_k), dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        N.check(N.lib().ojx_token_logprobs_workspace_bytes(rows, v, top_k, dt,
                                                           ctypes.byref(nbytes)),
                "token_logprobs_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        N.check(N.lib().ojx_token_logprobs(
            N.ptr(x), x.stride(0), rows, v, dt, N.ptr(tokens), top_k, N.ptr(lp), N.ptr(h),
            N.ptr(lse), N.ptr(stats), N.ptr(top), N.ptr(top_ids), N.ptr(ws), nbytes.value,
            N.stream_handle(dev)), "token_logprobs")
    s = logits.shape[:-1]
    return (lp.reshape(s), h.reshape(s), lse.reshape(s), top.reshape(*s, top_k),
            top_ids.reshape(*s, top_k), stats.reshape(*s, 2))


@token_logprobs.register_fake
def _(logits, ids, top_k):
    s = logits.shape[:-1]
    f = [logits.new_empty(s, dtype=torch.float32) for _ in range(3)]
    return (*f, logits.new_empty((*s, top_k), dtype=torch.float32),
            logits.new_empty((*s, top_k), dtype=torch.int64),
            logits.new_empty((*s, 2), dtype=torch.float32))


@torch.library.custom_op(f"{_NS}::token_logprobs_bwd", mutates_args=())
def token_logprobs_bwd(logits: torch.Tensor, ids: torch.Tensor, entropy: torch.Tensor,
                       stats: torch.Tensor, top_ids: torch.Tensor,
                       grad_logprob: Optional[torch.Tensor], grad_entropy: Optional[torch.Tensor],
                       grad_lse: Optional[torch.Tensor], grad_top: Optional[torch.Tensor]
                       ) -> torch.Tensor:
    """The logits' gradient from those of token_logprobs' results (None: zero)."""
    dev = N.require_device(logits, ids, entropy, stats, top_ids, grad_logprob, grad_entropy,
                           grad_lse, grad_top)
    dt = _dtype_code(logits.dtype)
    x, tokens = _logit_rows(logits, ids)
    rows, v = x.shape
    top_k = top_ids.shape[-1] if top_ids.dim() == ids.dim() + 1 else -1
    if top_ids.dtype != torch.int64 or top_ids.shape != (*ids.shape, top_k):
        raise RuntimeError(f"top_ids must be int64 [..., k] over {list(ids.shape)} "
                           f"(got {top_ids.dtype} {list(top_ids.shape)})")

    def rows_of(what, t, shape):
        if t is None:
            return None
        if t.dtype != torch.float32 or t.shape != shape:
            raise RuntimeError(f"{what} must be float32 {list(shape)} "
                               f"(got {t.dtype} {list(t.shape)})")
        return t.contiguous()

    h, s = rows_of("entropy", entropy, ids.shape), rows_of("stats", stats, (*ids.shape, 2))
    g = [rows_of("grad_logprob", grad_logprob, ids.shape),
         rows_of("grad_entropy", grad_entropy, ids.shape),
         rows_of("grad_lse", grad_lse, ids.shape), rows_of("grad_top", grad_top, top_ids.shape)]
    ti = top_ids.contiguous()
    gx = torch.empty((rows, v), dtype=logits.dtype, device=dev)
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_token_logprobs_bwd(
            N.ptr(x), x.stride(0), rows, v, dt, N.ptr(tokens), N.ptr(h), N.ptr(s), top_k,
            N.ptr(ti), *(N.ptr(t) for t in g), N.ptr(gx), N.stream_handle(dev)),
            "token_logprobs_bwd")
    return gx.reshape(logits.shape)


@token_logprobs_bwd.register_fake
def _(logits, ids, entropy, stats, top_ids, grad_logprob, grad_entropy, grad_lse, grad_top):
    return logits.new_empty(logits.shape)


def _logprobs_setup(ctx, inputs, output):
    logits, ids, _ = inputs
    _, entropy, _, _, top_ids, stats = output
    ctx.save_for_backward(logits, ids, entropy, stats, top_ids)
    ctx.mark_non_differentiable(top_ids, stats)
    ctx.set_materialize_grads(False)


def _logprobs_backward(ctx, g_lp, g_h, g_lse, g_top, *_):
    logits, ids, entropy, stats, top_ids = ctx.saved_tensors
    if not ctx.needs_input_grad[0] or (g_lp is None and g_h is None and g_lse is None
                                       and g_top is None):
        return None, None, None
    return token_logprobs_bwd(logits, ids, entropy, stats, top_ids, g_lp, g_h, g_lse, g_top), None, \
        None


token_logprobs.register_autograd(_logprobs_backward, setup_context=_logprobs_setup)


# ----------------------------------------------------------------------------- rotated positions

def _rotary_sizes(x: torch.Tensor) -> Tuple[int, int]:
    """(batches, tokens) of [tokens, heads, d] or [batch, tokens, heads, d]."""
    return (1, x.shape[0]) if x.dim() == 3 else (x.shape[0], x.shape[1])


def _rotary_input(x: torch.Tensor) -> torch.Tensor:
    """x as it lies, where the elements of a head are neighbours."""
    return x if x.stride(-1) == 1 else x.contiguous()


def _rotary_output(x: torch.Tensor) -> torch.Tensor:
    """As x lies, where that leaves a head's elements neighbours (not of heads that overlap in x)."""
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 else torch.empty_like(x, memory_format=torch.contiguous_format)


def _rotary_rows(x: torch.Tensor, y: torch.Tensor) -> "N.RotaryRows":
    return N.RotaryRows(N.ptr(x), N.ptr(y), x.stride(0) if x.dim() == 4 else 0, x.stride(-3),
                        x.stride(-2), y.stride(0) if x.dim() == 4 else 0, y.stride(-3),
                        y.stride(-2), x.shape[-2])


def _check_rotation(positions: torch.Tensor, shape: Tuple[int, ...], rates: torch.Tensor,
                    head_dim: int) -> Tuple[int, int]:
    """The positions' strides over batches and tokens."""
    if positions.dtype not in (torch.int32, torch.int64) or \
            tuple(positions.shape) not in (shape, shape[-1:]):
        raise RuntimeError(f"positions must be int32 or int64 {list(shape)} or {list(shape[-1:])} "
                           f"(got {positions.dtype} {list(positions.shape)})")
    if rates.dtype != torch.int64 or rates.dim() != 1 or not rates.is_contiguous():
        raise RuntimeError(f"rates must be contiguous int64 [pairs] "
                           f"(got {rates.dtype} {list(rates.shape)})")
    if not 1 <= rates.numel() <= head_dim // 2:
        raise RuntimeError(f"{rates.numel()} rotated pairs do not fit heads of {head_dim}")
    return (positions.stride(0) if positions.dim() == 2 else 0), positions.stride(-1)


@torch.library.custom_op(f"{_NS}::rotary", mutates_args=())
def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
           rates: torch.Tensor, gain: float, interleaved: bool, inverse: bool
           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """q and k (None: an empty tensor in its place) rotated, by the negative angles if inverse."""
    dev = N.require_device(q, k, positions, rates)
    dt = _dtype_code(q.dtype)
    if q.dim() not in (3, 4):
        raise RuntimeError("q must be [tokens, heads, head size] or [batch, tokens, heads, head size] "
                           f"(got {list(q.shape)})")
    lead, d = tuple(q.shape[:-2]), q.shape[-1]
    if k is not None and (k.dtype != q.dtype or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2]
                          or k.shape[-1] != d):
        raise RuntimeError(f"k must be {q.dtype} {[*lead, 'heads', d]} "
                           f"(got {k.dtype} {list(k.shape)})")
    pb, pt = _check_rotation(positions, lead, rates, d)
    rows, out = [], []
    for x in (q, k):
        if x is None:
            out.append(q.new_empty(0))
            continue
        x = _rotary_input(x)
        out.append(_rotary_output(x))
        rows.append((x, _rotary_rows(x, out[-1])))
    rot = N.Rotation(N.ptr(rates), rates.numel(), N.ptr(positions),
                     positions.dtype == torch.int64, interleaved, gain, inverse)
    with torch.cuda.device(dev):
        N.check(N.lib().ojx_rotary(
            ctypes.byref(rows[0][1]), ctypes.byref(rows[1][1]) if k is not None else None,
            *_rotary_sizes(q), d, dt, ctypes.byref(rot), pb, pt, N.stream_handle(dev)), "rotary")
    return out[0], out[1]


@rotary.register_fake
def _(q, k, positions, rates, gain, interleaved, inverse):
    return (_rotary_output(_rotary_input(q)),
            q.new_empty(0) if k is None else _rotary_output(_rotary_input(k)))


def _rotary_setup(ctx, inputs, output):
    _, k, positions, rates, gain, interleaved, inverse = inputs
    ctx.save_for_backward(positions, rates)
    ctx.rest = (gain, interleaved, not inverse)
    ctx.pair = k is not None
    ctx.set_materialize_grads(False)


def _rotary_backward(ctx, g_q, g_k):
    positions, rates = ctx.saved_tensors
    if not ctx.pair or not ctx.needs_input_grad[1]:
        g_k = None
    if not ctx.needs_input_grad[0]:
        g_q = None
    out = [None, None]
    if g_q is not None and g_k is not None:
        out = rotary(g_q, g_k, positions, rates, *ctx.rest)
    elif g_q is not None:
        out[0] = rotary(g_q, None, positions, rates, *ctx.rest)[0]
    elif g_k is not None:
        out[1] = rotary(g_k, None, positions, rates, *ctx.rest)[0]
    return out[0], out[1], None, None, None, None, None


rotary.register_autograd(_rotary_backward, setup_context=_rotary_setup)


# ----------------------------------------------------------------------------- beam search

@torch.library.custom_op(f"{_NS}::beam_select", mutates_args=())
def beam_select(logits: torch.Tensor, scores: torch.Tensor, num: int,
                finished: Optional[torch.Tensor], pad_id: int
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(scores, parents, tokens) [groups, num] of logits [groups, beams, V] and scores."""
    dev = N.require_device(logits, scores, finished)
    dt = _dtype_code(logits.dtype)
    if logits.dim() != 3 or logits.shape[2] < 1:
        raise RuntimeError(f"logits must be [groups, beams, vocabulary] (got {list(logits.shape)})")
    g, k, v = logits.shape
    if not 1 <= k <= MAX_BEAMS:
        raise RuntimeError(f"{k} beams, expected 1..{MAX_BEAMS}")
    if not 1 <= num <= min(MAX_TOP, k * v):
        raise RuntimeError(f"num is {num}, expected 1..{min(MAX_TOP, k * v)}")
    if scores.dtype != torch.float32 or tuple(scores.shape) != (g, k):
        raise RuntimeError(f"scores must be float32 {[g, k]} (got {scores.dtype} {list(scores.shape)})")
    if finished is not None:
        if finished.dtype != torch.bool or tuple(finished.shape) != (g, k):
            raise RuntimeError(f"finished must be bool {[g, k]} "
                               f"(got {finished.dtype} {list(finished.shape)})")
        if not 0 <= pad_id < v:
            raise RuntimeError(f"pad_id {pad_id} is outside the vocabulary of {v}")
        finished = finished.contiguous()
    x = logits.reshape(g * k, v)
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < v):
        x = x.contiguous()
    s = scores.contiguous()
    best = torch.empty((g, num), dtype=torch.float32, device=dev)
    parents = torch.empty((g, num), dtype=torch.int64, device=dev)
    tokens = torch.empty_like(parents)
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        N.check(N.lib().ojx_beam_select_workspace_bytes(g, k, v, num, dt, ctypes.byref(nbytes)),
                "beam_select_workspace_bytes")
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        N.check(N.lib().ojx_beam_select(
            N.ptr(x), x.stride(0), g, k, v, dt, N.ptr(s), N.ptr(finished), pad_id, num, N.ptr(best),
            N.ptr(parents), N.ptr(tokens), N.ptr(ws), nbytes.value, N.stream_handle(dev)),
            "beam_select")
    return best, parents, tokens


@beam_select.register_fake
def _(logits, scores, num, finished, pad_id):
    shape = (logits.shape[0], num)
    return (scores.new_empty(shape), scores.new_empty(shape, dtype=torch.int64),
            scores.new_empty(shape, dtype=torch.int64))
