"""Plain forms of the 8-bit paged cache, its attention and token log probabilities, for tests:
element by element from the definitions, in 64 bits but where the cache's own arithmetic is
32-bit (scales and codes)."""

import math

import numpy as np
import torch


def stored(d):
    return (d + 63) // 64 * 64


def key_byte(t, d, dp):
    """Byte of key d of token t within its block and head."""
    g, t = divmod(t, 16)
    return g * 16 * dp + (d // 64) * 1024 + (t // 4) * 256 + (d % 64 // 16) * 64 + (t % 4) * 16 + d % 16


def value_byte(t, d, dp):
    g, t = divmod(t, 16)
    return g * 16 * dp + d * 16 + t


def byte_maps(block, dp):
    """(keys', values') byte of every (token, d), as [block, dp] arrays."""
    t, d = np.meshgrid(np.arange(block), np.arange(dp), indexing="ij")
    return key_byte(t, d, dp), value_byte(t, d, dp)


def codes_of(cache):
    """The cache's codes as [blocks, heads, token, d] int arrays (keys, values)."""
    n, h, b, dp = cache.k_codes.shape
    km, vm = byte_maps(b, dp)
    k = cache.k_codes.cpu().numpy().reshape(n, h, -1)[:, :, km]
    v = cache.v_codes.cpu().numpy().reshape(n, h, -1)[:, :, vm]
    return k.astype(np.int64), v.astype(np.int64)


def fill(cache, generator, width=40.0):
    """Random codes in every stored byte (padding too) and positive scales."""
    for t in (cache.k_codes, cache.v_codes):
        x = torch.randn(t.shape, generator=generator) * width
        t.copy_(x.round().clamp(-127, 127).to(torch.int8))
    s = 0.02 * torch.exp(0.5 * torch.randn(cache.scales.shape, generator=generator))
    cache.scales.copy_(s)


def plan(seq, new, tables, free, num_free, block, tokens):
    """(tables, slots, positions, requests, starts, lens, left) by loops over tokens."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    slots, positions, requests, starts, lens = [], [], [], [0], []
    top = min(num_free, len(free))
    for r, (s, n) in enumerate(zip(seq, new)):
        s, n = max(s, 0), max(n, 0)
        n = min(n, tokens - len(slots))
        for p in range(s, s + n):
            j = p // block
            if p % block == 0 and j < width:
                top -= 1
                tables[r][j] = free[top] if top >= 0 else -1
            e = tables[r][j] if j < width else -1
            slots.append(e * block + p % block if e >= 0 else -1)
            positions.append(p)
            requests.append(r)
        starts.append(len(slots))
        lens.append(s + n)
    pad = [-1] * (tokens - len(slots))
    return tables, slots + pad, positions + pad, requests + pad, starts, lens, top


def append(codes, scales, x, slots, block):
    """x [tokens, heads, d] float32 into codes [blocks, heads, token, dp], scales [blocks, heads]
    in place: one block after another, in 32-bit arithmetic as the cache defines it."""
    f32 = np.float32
    blocks, heads, _, _ = codes.shape
    d = x.shape[2]
    runs, last = [], None
    for t, s in enumerate(slots):
        if not 0 <= s < blocks * block:
            last = None
            continue
        if last is not None and s == last + 1 and s % block:
            runs[-1].append(t)
        else:
            runs.append([t])
        last = s
    for run in runs:
        b, off = divmod(int(slots[run[0]]), block)
        for h in range(heads):
            e = x[run, h].astype(f32)
            a = np.abs(e[np.isfinite(e)])
            m = f32(a.max()) if a.size else f32(0)
            m = m if m >= f32(2.0) ** -100 else f32(0)
            before = scales[b, h] if off else f32(0)
            s = max(before, f32(m * f32(1 / 127)))
            with np.errstate(all="ignore"):
                inv = f32(1) / s if s > 0 else f32(0)
                if off and s > before:
                    old = codes[b, h, :off].astype(f32) * (before / s)
                    codes[b, h, :off] = np.rint(old).astype(np.int64)
                c = np.rint(e * inv)
                c = np.where(np.isnan(c), 0, np.clip(c, -127, 127))
            codes[b, h, off:off + len(run), :d] = c.astype(np.int64)
            scales[b, h] = s


def attention(q, k, v, k_scale, v_scale, tables, lens, starts, scale, window, block):
    """(out, lse, bound of the scores' error per unit of q's rounding) in float64: q [tokens,
    heads, d]; k, v codes [blocks, kv heads, token, dp]."""
    t, hq, d = q.shape
    nb, hkv = k.shape[:2]
    out, lse = np.zeros((t, hq, d)), np.full((t, hq), -np.inf)
    reach = np.zeros((t, hq))  # largest sum_d |k_d| of a visible key
    vmax = np.zeros((t, hq))
    for r in range(len(lens)):
        for i in range(starts[r], starts[r + 1]):
            pos = lens[r] - (starts[r + 1] - starts[r]) + i - starts[r]
            lo = max(0, pos + 1 - window) if window else 0
            js = [j for j in range(lo, pos + 1)
                  if j // block < len(tables[r]) and 0 <= tables[r][j // block] < nb]
            if not js:
                continue
            b = np.array([tables[r][j // block] for j in js])
            o = np.array([j % block for j in js])
            for h in range(hq):
                g = h // (hq // hkv)
                kk = k[b, g, o, :d] * k_scale[b, g][:, None].astype(np.float64)
                vv = v[b, g, o, :d] * v_scale[b, g][:, None].astype(np.float64)
                s = kk @ q[i, h].astype(np.float64) * scale
                m = s.max()
                p = np.exp(s - m)
                out[i, h] = p @ vv / p.sum()
                lse[i, h] = m + math.log(p.sum())
                reach[i, h] = np.abs(kk).sum(1).max()
                vmax[i, h] = 127 * v_scale[b, g].max()
    return out, lse, reach, vmax


def logprobs(x, ids, top):
    """(logprob, entropy, lse, top, top_ids, log p) of float64 rows, -inf allowed."""
    m = x.max(1, keepdims=True)
    base = np.where(np.isneginf(m), 0.0, m)
    e = np.exp(x - base)
    with np.errstate(divide="ignore", invalid="ignore"):
        ls = np.log(e.sum(1))
        lse = ls + base[:, 0]
        # not x - lse: beside the lowest value of a type even 64 bits have no room for log s
        logp = np.where(np.isneginf(x), -np.inf, (x - base) - ls[:, None])
    p = np.exp(logp)
    h = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(1)
    v = x.shape[1]
    lp = np.array([logp[i, j] if 0 <= j < v else 0.0 for i, j in enumerate(ids)])
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return lp, h, lse, np.take_along_axis(logp, order, 1), order, logp
