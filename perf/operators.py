"""Performance cases of the serving and training operators around the packed linears.

* ``plan``: the block tables and slot maps of a batch's next step, from its requests' lengths;
* ``append``: keys and values of new tokens into an 8-bit paged cache with one scale for each
  block of tokens and head, and the touched blocks read back as values;
* ``attention``: causal attention of the newest tokens over that cache, paged, grouped heads;
* ``logprobs``: log probabilities of given tokens with entropy and the top alternatives, for
  answers; ``logprobs_train``: the same with the gradient of the logits.

Cache layout (what ``prepare`` makes): codes are int8 ``[blocks, kv heads, block, Dp]`` with Dp
the head size rounded up to 64.  Inside one block and head, 16 tokens at a time, keys lie as
``[Dp/64][4][4][4][16]`` = (d / 64, token / 4, d % 64 / 16, token % 4, d % 16) and values as
``[Dp][16]`` = (d, token).  ``scales`` is fp32 ``[blocks, kv heads, 2]``: keys, values.
"""

import math
import os
import random
import sys

import torch

own = False

DEV = torch.device("cuda:0")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    path = os.path.abspath("ojasx-open-source-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ojasx_amd

    return ojasx_amd


def listed():
    return [
        # the next step of 64 requests that each generate one token: launch latency
        {"name": "plan_decode_64", "kind": "plan", "r": 64, "ctx_lo": 10, "ctx_hi": 4000,
         "new_hi": 1, "prompts": 0.0, "block": 64},
        # a large scheduler step: 4096 requests, one in twenty with a prompt of up to 2000 tokens
        {"name": "plan_mixed_4096", "kind": "plan", "r": 4096, "ctx_lo": 1, "ctx_hi": 8000,
         "new_hi": 2000, "prompts": 0.05, "block": 32},
        # one new token for each of 64 requests, written into partly filled blocks
        {"name": "append_decode_64", "kind": "append", "r": 64, "ctx_lo": 10, "ctx_hi": 4000,
         "new_lo": 1, "new_hi": 1, "hkv": 8, "d": 128, "block": 64, "dtype": "bf16"},
        # the prompts of seven requests in one step, ragged, in small blocks
        {"name": "append_prompts_fp16", "kind": "append", "r": 7, "ctx_lo": 1, "ctx_hi": 500,
         "new_lo": 500, "new_hi": 6000, "hkv": 8, "d": 80, "block": 16, "dtype": "fp16"},
        # one user's token over a conversation of about two thousand tokens: latency
        {"name": "attend_one", "kind": "attention", "r": 1, "ctx_lo": 2047, "ctx_hi": 2047,
         "new_lo": 1, "new_hi": 1, "hq": 32, "hkv": 8, "d": 128, "block": 64, "window": 0,
         "dtype": "bf16"},
        # a full decode batch over ragged contexts: the cache streams from memory
        {"name": "attend_batch_64", "kind": "attention", "r": 64, "ctx_lo": 500, "ctx_hi": 16000,
         "new_lo": 1, "new_hi": 1, "hq": 32, "hkv": 8, "d": 128, "block": 64, "window": 0,
         "dtype": "bf16"},
        # chunks of long prompts over what is cached of them: products bound it
        {"name": "attend_prompt_chunks", "kind": "attention", "r": 4, "ctx_lo": 1000,
         "ctx_hi": 6000, "new_lo": 900, "new_hi": 2048, "hq": 32, "hkv": 8, "d": 128, "block": 64,
         "window": 0, "dtype": "bf16"},
        # drafts of one to five tokens to be verified: one head group of one, odd head size,
        # small blocks, a sliding window, a request without any context
        {"name": "attend_drafts_fp16", "kind": "attention", "r": 9, "ctx_lo": 0, "ctx_hi": 3000,
         "new_lo": 1, "new_hi": 5, "hq": 20, "hkv": 20, "d": 80, "block": 16, "window": 1000,
         "dtype": "fp16"},
        # a decode step's answer: sampled tokens of 8 requests with 8 alternatives each
        {"name": "answer_8", "kind": "logprobs", "t": 8, "v": 128256, "top": 8, "masked": 0.0,
         "dtype": "bf16"},
        # constrained decoding in fp32: most of an odd vocabulary masked, some tokens not asked for
        {"name": "answer_masked_fp32", "kind": "logprobs", "t": 77, "v": 50021, "top": 20,
         "masked": 0.9, "dtype": "fp32"},
        # scoring of a batch of sequences against a smaller vocabulary
        {"name": "score_4096_fp16", "kind": "logprobs", "t": 4096, "v": 32000, "top": 5,
         "masked": 0.0, "dtype": "fp16"},
        # a policy step: log probabilities and entropy of 2048 tokens and the logits' gradient
        {"name": "policy_2048", "kind": "logprobs_train", "t": 2048, "v": 128256, "top": 0,
         "masked": 0.0, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["plan", "append", "append", "attention", "attention", "attention",
                       "logprobs", "logprobs_train"])
    if kind == "plan":
        return {"kind": kind, "r": log(1, 4096), "ctx_lo": 1, "ctx_hi": log(50, 8000),
                "new_hi": log(1, 2000), "prompts": rng.choice([0.0, 0.02, 0.05]),
                "block": rng.choice([16, 32, 64, 128])}
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind in ("append", "attention"):
        d = rng.choice([64, 80, 96, 128, 128, 192, 256])
        hkv = rng.choice([1, 2, 4, 5, 8, 8])
        case = {"kind": kind, "r": log(1, 64), "ctx_lo": rng.choice([0, 1, 100]),
                "ctx_hi": log(200, 16000), "hkv": hkv, "d": d,
                "block": rng.choice([16, 32, 64, 128]), "dtype": dtype}
        # generation, drafts, or prompts
        case["new_lo"], case["new_hi"] = rng.choice([(1, 1), (1, rng.randint(2, 9)),
                                                     (rng.randint(20, 100), log(100, 2048))])
        if kind == "append":
            while _tokens(case) * hkv * d > 17000 * 8 * 128:
                case["r"] = max(1, case["r"] // 2)
            return case
        case["hq"] = hkv * rng.choice([1, 2, 4, 4, 7, 8])
        case["window"] = rng.choice([0, 0, 0, log(64, 4000)])
        while case["r"] > 1 and (work(case)["flops"] > 3e11 or _padded(case) > 3e9):
            case["r"] //= 2
        while work(case)["flops"] > 3e11 or _padded(case) > 3e9:
            case["hq"] = case["hkv"] = 1
            case["new_hi"] = max(case["new_lo"], case["new_hi"] // 2)
        return case
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    v = log(1000, 130000)
    t = log(1, 4096)
    while t * v > 2048 * 128256:
        t //= 2
    return {"kind": kind, "t": t, "v": v, "top": rng.choice([0, 1, 5, 8, 20]),
            "masked": rng.choice([0.0, 0.0, 0.5]), "dtype": dtype}


# ------------------------------------------------------------------ sizes of a case

def _lens(case):
    """(context, new tokens) of each request: ragged, of the case alone."""
    rng = random.Random(case["r"] * 1_000_003 + case["ctx_hi"] * 101 + case["new_hi"])
    lo, hi = max(1, case["ctx_lo"]), max(1, case["ctx_hi"])
    ctx = [int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) for _ in range(case["r"])]
    if case["ctx_lo"] == 0:
        ctx[0] = 0
    if case["kind"] == "plan":
        new = [rng.randint(1, case["new_hi"]) if rng.random() < case["prompts"] else 1
               for _ in range(case["r"])]
    else:
        new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["r"])]
    return ctx, new


def _tokens(case):
    return sum(_lens(case)[1])


def _padded(case):
    """Scores and keys of the padded batch that the plain form works on."""
    ctx, new = _lens(case)
    longest = max(c + n for c, n in zip(ctx, new))
    return case["r"] * longest * max(case["hq"] * max(new), case["hkv"] * case["d"])


def _visible(c, n, window):
    """Keys that the n newest tokens after c others see, summed over the tokens."""
    if not window:
        return n * c + n * (n + 1) // 2
    return sum(min(c + i + 1, window) for i in range(n))


def work(case):
    kind = case["kind"]
    if kind == "plan":
        ctx, new = _lens(case)
        b = case["block"]
        blocks = sum(-(-(c + n) // b) - -(-c // b) for c, n in zip(ctx, new))
        # lengths, tables' last entries, new blocks from the stack to the tables; per token its
        # slot, position and request
        return {"bytes": case["r"] * 20 + blocks * 8 + sum(new) * 16, "flops": 0}
    if kind == "append":
        ctx, new = _lens(case)
        b, hd = case["block"], case["hkv"] * case["d"]
        touched = sum(-(-(c + n) // b) - c // b for c, n in zip(ctx, new))
        held = sum(c + n - c // b * b for c, n in zip(ctx, new))
        size = SIZE[case["dtype"]]
        # new keys and values in, their codes out; codes of the touched blocks in, values out
        return {"bytes": 2 * hd * (sum(new) * (size + 1) + held + touched * b * size)
                + touched * case["hkv"] * 16, "flops": 0}
    if kind == "attention":
        ctx, new = _lens(case)
        w, hd = case["window"], case["hkv"] * case["d"]
        seen = sum(min(c + n, w + n - 1) if w else c + n for c, n in zip(ctx, new))
        q = sum(new) * case["hq"] * case["d"]
        pairs = sum(_visible(c, n, w) for c, n in zip(ctx, new))
        return {"bytes": 2 * seen * hd + seen // case["block"] * case["hkv"] * 8
                + 2 * q * SIZE[case["dtype"]], "flops": 4 * pairs * case["hq"] * case["d"]}
    n = case["t"] * case["v"] * SIZE[case["dtype"]]
    return {"bytes": (3 if kind == "logprobs_train" else 1) * n + case["t"] * (16 + 12 * case["top"]),
            "flops": 0}


# ------------------------------------------------------------------ inputs

def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (salt + 1) + seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(case, held, seed):
    """Random block tables for `held` tokens of each request, and the rest of the pool."""
    b = case["block"]
    need = [-(-h // b) for h in held]
    ctx, new = _lens(case)
    width = max(1, max(-(-(c + n) // b) for c, n in zip(ctx, new))) + 2
    total = sum(-(-(c + n) // b) for c, n in zip(ctx, new)) + 5
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
    tables = torch.full((case["r"], width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = perm[at:at + n]
        at += n
    return tables.to(DEV), perm[at:].to(torch.int32).to(DEV), total


def prepare(case, seed):
    kind = case["kind"]
    state = {"case": case}
    if kind in ("logprobs", "logprobs_train"):
        g = _gen(seed)
        t, v, dt = case["t"], case["v"], DTYPES[case["dtype"]]
        # logits of a model: a broad spread with a few likely tokens in each row
        x = torch.randn(t, v, generator=g, device=DEV, dtype=torch.float32).mul_(2.0)
        likely = torch.randint(0, v, (t, 10), generator=g, device=DEV)
        x.scatter_add_(1, likely, torch.rand(t, 10, generator=g, device=DEV) * 12)
        if case["masked"]:
            x.masked_fill_(torch.rand(t, v, generator=g, device=DEV) < case["masked"], -math.inf)
        ids = torch.where(torch.rand(t, generator=g, device=DEV) < 0.7, likely[:, 0],
                          torch.randint(0, v, (t,), generator=g, device=DEV))
        ids[torch.rand(t, generator=g, device=DEV) < 0.05] = -100  # tokens not asked for
        if case["masked"]:
            # an asked token is an allowed one
            x.scatter_(1, ids.clamp(min=0)[:, None], 1.5)
        state.update(x=x.to(dt), ids=ids)
        if kind == "logprobs_train":
            state["x"].requires_grad_(True)
            state["g_lp"] = torch.randn(t, generator=g, device=DEV)
            state["g_h"] = torch.randn(t, generator=g, device=DEV) * 0.1
            state["g_top"] = torch.randn(t, case["top"], generator=g, device=DEV)
        return state

    ctx, new = _lens(case)
    if kind == "plan":
        tables, free, _ = _tables(case, ctx, seed)
        state.update(tables=tables, free=free, num_free=_i32([free.numel()]), ctx=_i32(ctx),
                     new=_i32(new), t=sum(new))
        return state

    g = _gen(seed, 1)
    tables, _, total = _tables(case, [c + n for c, n in zip(ctx, new)], seed)
    b, h, d, dt = case["block"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    dp = -(-d // 64) * 64
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    shape = (total, h, b, dp)
    for name in ("k_codes", "v_codes"):
        codes = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
        state[name] = codes.mul_(35).round_().clamp_(-127, 127).to(torch.int8)
        del codes
    # a block's scale: its largest value over 127, about 3.5 deviations, more in some blocks
    scales = (3.6 / 127) * torch.exp(0.25 * torch.randn(total, h, 2, generator=g, device=DEV))
    state.update(scales=scales.float(), tables=tables)
    if kind == "attention":
        if dp > d:  # the stored head size is padded with zeros
            state["v_codes"].view(total, h, b // 16, dp, 16)[:, :, :, d:] = 0
            state["k_codes"].copy_(_k_in(_k_out(state["k_codes"]).mul_(
                (torch.arange(dp, device=DEV) < d).to(torch.int8))))
        q = torch.randn(sum(new), case["hq"], d, generator=g, device=DEV).mul_(1.5)
        state.update(q=q.to(dt), lens=_i32([c + n for c, n in zip(ctx, new)]),
                     starts=None if case["new_hi"] == 1 else _i32(starts), longest=max(
                         c + n for c, n in zip(ctx, new)), newest=max(new))
        return state
    # keys with some large channels, as keys have
    wide = 1 + 3 * (torch.arange(d, device=DEV) % 17 == 5).float()
    state["k"] = (torch.randn(sum(new), h, d, generator=g, device=DEV) * wide).to(dt)
    state["v"] = torch.randn(sum(new), h, d, generator=g, device=DEV).to(dt)
    req = torch.repeat_interleave(torch.arange(case["r"]), torch.tensor(new))
    pos = torch.arange(sum(new)) - torch.tensor(starts)[req] + torch.tensor(ctx)[req]
    tab = tables.cpu().long()
    state["slots"] = (tab[req, pos // b] * b + pos % b).to(DEV)
    state["blocks"] = torch.cat([tab[r, c // b:-(-(c + n) // b)]
                                 for r, (c, n) in enumerate(zip(ctx, new))]).to(torch.int32).to(DEV)
    return state


# ------------------------------------------------------------------ plain forms

def _k_out(codes):
    """Keys of the cache as [blocks, heads, token, d]."""
    n, h, b, dp = codes.shape
    x = codes.view(n, h, b // 16, dp // 64, 4, 4, 4, 16).permute(0, 1, 2, 4, 6, 3, 5, 7)
    return x.reshape(n, h, b, dp)


def _k_in(x):
    """The inverse of _k_out, in the cache's shape."""
    n, h, b, dp = x.shape
    x = x.view(n, h, b // 16, 4, 4, dp // 64, 4, 16).permute(0, 1, 2, 5, 3, 6, 4, 7)
    return x.reshape(n, h, b, dp)


def _v_out(codes):
    n, h, b, dp = codes.shape
    return codes.view(n, h, b // 16, dp, 16).transpose(3, 4).reshape(n, h, b, dp)


def _v_in(x):
    n, h, b, dp = x.shape
    return x.view(n, h, b // 16, 16, dp).transpose(3, 4).reshape(n, h, b, dp)


def _plain_plan(s):
    b, tables = s["case"]["block"], s["tables"]
    r, w = tables.shape
    old, new = s["ctx"], s["new"]
    have = ((old + b - 1) // b).clamp(max=w)
    want = ((old + new + b - 1) // b).clamp(max=w)
    need = want - have
    ends = torch.cumsum(need, 0)
    col = torch.arange(w, device=DEV)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    at = s["num_free"] - 1 - ((ends - need)[:, None] + col - have[:, None])
    got = s["free"][at.clamp(0, s["free"].numel() - 1)]
    tables.copy_(torch.where(fresh, torch.where(at >= 0, got, -1), tables))
    starts = torch.zeros(r + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum(new, 0)
    t = torch.arange(s["t"], device=DEV, dtype=torch.int32)
    req = torch.searchsorted(starts[1:].contiguous(), t, right=True).to(torch.int32)
    pos = old[req] + t - starts[req]
    block = tables[req, pos // b].long()
    slots = torch.where(block >= 0, block * b + pos % b, -1)
    return {"tables": tables, "slots": slots, "positions": pos, "requests": req, "starts": starts,
            "lens": old + new, "num_free": (s["num_free"] - ends[-1]).to(torch.int32)}


def _plain_append(s):
    case, slots, scales = s["case"], s["slots"], s["scales"]
    b, d, dt = case["block"], case["d"], DTYPES[case["dtype"]]
    block, off = slots // b, slots % b
    # the first new token of every touched block, and which touched block a token is in
    touched = s["blocks"].long()
    place = torch.zeros(scales.shape[0], dtype=torch.int64, device=DEV)
    place[touched] = torch.arange(touched.numel(), device=DEV)
    run = place[block]
    first = torch.full((touched.numel(),), b, device=DEV)
    first = first.scatter_reduce(0, run, off, "amin")
    tok = torch.arange(b, device=DEV)
    out = []
    for i, (x, codes, out_of, into) in enumerate(((s["k"], s["k_codes"], _k_out, _k_in),
                                                  (s["v"], s["v_codes"], _v_out, _v_in))):
        x = x.float()
        amax = torch.zeros(touched.numel(), x.shape[1], device=DEV)
        amax = amax.scatter_reduce(0, run[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        before = torch.where(first[:, None] > 0, scales[touched, :, i], 0)
        scale = torch.maximum(before, amax * (1.0 / 127))
        old = out_of(codes[touched]).float()
        ratio = torch.where(scale > 0, before / scale, 0)[:, :, None, None]
        kept = (tok < first[:, None])[:, None, :, None]
        now = torch.where(kept, torch.round(old * ratio), old)
        inverse = torch.where(scale > 0, 1 / scale, 0)
        code = torch.round(x * inverse[run][:, :, None]).clamp(-127, 127)
        now[run, :, off, :d] = code
        codes[touched] = into(now.to(torch.int8))
        scales[touched, :, i] = scale
        out.append((now[..., :d] * scale[:, :, None, None]).transpose(1, 2).to(dt).contiguous())
    return {"k": out[0], "v": out[1], "scales": scales[touched]}


def _plain_attention(s):
    case, q, tables, lens = s["case"], s["q"], s["tables"], s["lens"]
    b, d, hkv, w = case["block"], case["d"], case["hkv"], case["window"]
    t, hq, _ = q.shape
    r, longest, newest = lens.numel(), s["longest"], s["newest"]
    starts = s["starts"]
    if starts is None:
        starts = torch.arange(r + 1, device=DEV, dtype=torch.int32)
    new = starts[1:] - starts[:-1]
    width = -(-longest // b)
    used = tables[:, :width].clamp(min=0).long()

    def dense(codes, i, out_of):
        x = out_of(codes)[..., :d].float() * s["scales"][:, :, i, None, None]
        x = x[used]  # [r, width, hkv, b, d]
        return x.transpose(1, 2).reshape(r, hkv, width * b, d)

    # queries padded to the longest, heads of a group beside each other
    i = torch.arange(newest, device=DEV)
    at = (starts[:-1, None] + i).clamp(max=t - 1).long()
    qp = q[at].float().mul(1 / math.sqrt(d)).view(r, newest, hkv, hq // hkv, d)
    qp = qp.permute(0, 2, 3, 1, 4).reshape(r, hkv, -1, d)
    scores = torch.matmul(qp, dense(s["k_codes"], 0, _k_out).transpose(2, 3))
    j = torch.arange(width * b, device=DEV)
    pos = (lens - new)[:, None] + i
    seen = j <= pos[:, :, None]
    if w:
        seen = seen & (j > pos[:, :, None] - w)
    seen = seen[:, None, None].expand(r, hkv, hq // hkv, -1, -1).reshape(r, hkv, -1, width * b)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, dense(s["v_codes"], 1, _v_out)) / total.clamp(min=1e-30)
    o = o.view(r, hkv, hq // hkv, newest, d).permute(0, 3, 1, 2, 4).reshape(r, newest, hq, d)
    return o[i < new[:, None]].to(q.dtype)


def _plain_logprobs(s):
    case, ids = s["case"], s["ids"]
    with torch.no_grad():
        x = s["x"].float()
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(m > -math.inf, m, 0))
        total = e.sum(-1, keepdim=True)
        lse = m + torch.log(total)
        logp = torch.where(x > -math.inf, x - lse, -math.inf)
        p = e / total.clamp(min=1e-30)
        h = -torch.where(p > 0, p * logp, 0).sum(-1)
        asked = (ids >= 0) & (ids < case["v"])
        at = ids.clamp(0, case["v"] - 1)[:, None]
        lp = torch.where(asked, logp.gather(1, at)[:, 0], 0)
        out = {"logprob": lp, "entropy": h}
        if case["top"]:
            # equal logits in the order of their tokens
            order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]
            out.update(top=logp.gather(1, order), top_ids=order)
        if case["kind"] == "logprobs_train":
            weight = torch.where(asked, s["g_lp"], 0)
            total_g = weight + s["g_top"].sum(-1)
            g = -p * (total_g[:, None] + s["g_h"][:, None]
                      * torch.where(p > 0, logp + h[:, None], 0))
            g.scatter_add_(1, at, weight[:, None])
            if case["top"]:
                g.scatter_add_(1, order, s["g_top"])
            out["grad"] = g.to(s["x"].dtype)
        return out


# ------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention,
                "logprobs": _plain_logprobs, "logprobs_train": _plain_logprobs}[kind](s)
    amd = _package()
    if kind == "plan":
        p = amd.kv8.plan(s["ctx"], s["new"], s["tables"], s["free"], s["num_free"],
                         s["case"]["block"], s["t"])
        return {"tables": s["tables"], "slots": p.slots, "positions": p.positions,
                "requests": p.requests, "starts": p.query_starts, "lens": p.seq_lens,
                "num_free": p.num_free}
    if kind == "append":
        amd.kv8.append(s["k"], s["v"], s["slots"], s["k_codes"], s["v_codes"], s["scales"])
        k, v, scales = amd.kv8.read(s["k_codes"], s["v_codes"], s["scales"], s["blocks"],
                                    s["case"]["d"], s["k"].dtype)
        return {"k": k, "v": v, "scales": scales}
    if kind == "attention":
        return amd.kv8.attention(s["q"], s["k_codes"], s["v_codes"], s["scales"], s["tables"],
                                 s["lens"], s["starts"], window=s["case"]["window"],
                                 max_query_len=s["newest"], max_seq_len=s["longest"])
    lp = amd.token_logprobs(s["x"], s["ids"], top_k=s["case"]["top"])
    out = {"logprob": lp.logprob, "entropy": lp.entropy}
    if s["case"]["top"]:
        out.update(top=lp.top_logprobs, top_ids=lp.top_ids)
    if kind == "logprobs_train":
        outs, grads = [lp.logprob, lp.entropy], [s["g_lp"], s["g_h"]]
        if s["case"]["top"]:
            outs.append(lp.top_logprobs)
            grads.append(s["g_top"])
        out["grad"], = torch.autograd.grad(outs, [s["x"]], grads)
        out = {k: v.detach() for k, v in out.items()}
    return out


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None
    b = case.get("block")
    if kind == "append":
        d, n = case["d"], s["blocks"].numel()
        where = {int(k): i for i, k in enumerate(s["blocks"].tolist())}
        slots = s["slots"].cpu()
        run_of = torch.tensor([where[int(x)] for x in (slots // b).tolist()], device=DEV)
        off = (slots % b).to(DEV)
        out, new_scales = [], []
        for i, (name, codes) in enumerate((("k", s["k_codes"]), ("v", s["v_codes"]))):
            raw = codes[s["blocks"].long()]
            dp = raw.shape[-1]
            tok = torch.arange(b, device=DEV)[:, None]
            dd = torch.arange(dp, device=DEV)[None, :]
            if name == "k":
                at = (tok // 16 * dp * 16 + dd // 64 * 1024 + tok % 16 // 4 * 256
                      + dd % 64 // 16 * 64 + tok % 4 * 16 + dd % 16)
            else:
                at = tok // 16 * dp * 16 + dd * 16 + tok % 16
            values = raw.reshape(n, -1, b * dp)[:, :, at].double()
            x = s[name].double()
            scale = torch.zeros(n, x.shape[1], device=DEV, dtype=torch.float64)
            first = torch.full((n,), b, device=DEV)
            first.scatter_reduce_(0, run_of, off, "amin")
            scale.scatter_reduce_(0, run_of[:, None].expand(-1, x.shape[1]), x.abs().amax(2) / 127,
                                  "amax")
            was = s["scales"][s["blocks"].long(), :, i].double() * (first > 0)[:, None]
            scale = torch.maximum(scale, was)
            keep = (torch.arange(b, device=DEV) < first[:, None])[:, None, :, None]
            values = torch.where(keep, torch.round(values * (was / scale)[:, :, None, None]), values)
            values[run_of, :, off, :d] = torch.round(x / scale[run_of][:, :, None])
            out.append((values[..., :d] * scale[:, :, None, None]).transpose(1, 2).contiguous())
            new_scales.append(scale)
        return {"k": out[0], "v": out[1], "scales": torch.stack(new_scales, -1)}
    if kind == "attention":
        ctx, new = _lens(case)
        hkv, g, d, w = case["hkv"], case["hq"] // case["hkv"], case["d"], case["window"]
        rows, first = [], 0
        for r, (c, n) in enumerate(zip(ctx, new)):
            used = s["tables"][r, :-(-(c + n) // b)].long()
            sc = s["scales"][used].double()
            k = (_k_out(s["k_codes"][used]).double() * sc[:, :, 0, None, None])[..., :d]
            v = (_v_out(s["v_codes"][used]).double() * sc[:, :, 1, None, None])[..., :d]
            k = k.transpose(0, 1).reshape(hkv, -1, d)[:, :c + n]
            v = v.transpose(0, 1).reshape(hkv, -1, d)[:, :c + n]
            q = s["q"][first:first + n].double().view(n, hkv, g, d)
            pos = torch.arange(c, c + n, device=DEV)[:, None]
            j = torch.arange(c + n, device=DEV)
            hide = (j > pos) | (j <= pos - w) if w else j > pos
            heads = []
            for i in range(hkv):
                a = q[:, i].transpose(0, 1).reshape(g * n, d) @ k[i].T / math.sqrt(d)
                a = torch.softmax(a.view(g, n, -1).masked_fill(hide, -math.inf), -1)
                heads.append((a.reshape(g * n, -1) @ v[i]).view(g, n, d).transpose(0, 1))
            rows.append(torch.cat(heads, 1))
            first += n
        return torch.cat(rows)
    out = {k: [] for k in ("logprob", "entropy") + (("top", "top_ids") if case["top"] else ())
           + (("grad",) if kind == "logprobs_train" else ())}
    for i in range(0, case["t"], 512):
        part = slice(i, i + 512)
        x = s["x"].detach()[part].double()
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        ids = s["ids"][part]
        asked = ids >= 0
        at = ids.clamp(min=0)[:, None]
        plogp = torch.where(p > 0, p * logp, 0)
        h = -plogp.sum(-1)
        out["logprob"].append(torch.where(asked, logp.gather(1, at)[:, 0], 0))
        out["entropy"].append(h)
        if case["top"]:
            order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
            out["top"].append(logp.gather(1, order))
            out["top_ids"].append(order)
        if kind == "logprobs_train":
            weight = s["g_lp"][part].double() * asked
            top = s["g_top"][part].double()
            g = -(p * (weight + top.sum(-1))[:, None]
                  + (plogp + p * h[:, None]) * s["g_h"][part].double()[:, None])
            g.scatter_add_(1, at, weight[:, None])
            if case["top"]:
                g.scatter_add_(1, order, top)
            out["grad"].append(g)
    return {k: torch.cat(v) for k, v in out.items()}
