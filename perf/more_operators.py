"""Performance cases of the operators of a decoding and a training step around the cache.

* ``rotary``: positions rotated into queries and keys; ``rotary_train``: with their gradients;
* ``append``: one call that rotates a step's queries and keys and writes keys and values into the
  8-bit paged cache, and the touched blocks read back as values;
* ``beam``: the best continuations of each group of beams over its beams and the vocabulary;
* ``reorder``: block tables, lengths and the stack of free blocks after beams were chosen, and the
  copies of begun blocks in every layer's cache.

Rotation: pair i of a head's first ``rot`` elements, (i, i + rot / 2) or interleaved (2 i, 2 i + 1),
turns by position times frequency; frequencies ``base ** (-2 i / rot)``, scaled for long contexts.

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
PAD = 2  # the token of a finished beam


def _package():
    path = os.path.abspath("ojasx-open-source-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ojasx_amd

    return ojasx_amd


def listed():
    return [
        # queries and keys of a decode batch of 64 requests: launch latency
        {"name": "rotary_decode_64", "kind": "rotary", "b": 1, "s": 64, "hq": 32, "hkv": 8, "d": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "far": 8000, "dtype": "bf16"},
        # scoring of one long document's end in fp32: far positions, frequencies scaled by parts,
        # a part of an odd head, neighbouring pairs
        {"name": "rotary_far_fp32", "kind": "rotary", "b": 1, "s": 777, "hq": 20, "hkv": 20, "d": 80,
         "rot": 32, "interleaved": True, "scaling": "ramp", "far": 1000000, "dtype": "fp32"},
        # a training step's layer: 4 sequences of 2048 tokens, grouped heads
        {"name": "rotary_train_8192", "kind": "rotary_train", "b": 4, "s": 2048, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "interleaved": False, "scaling": "none", "far": 0, "dtype": "bf16"},
        # fine-tuning on one sequence of odd length, a third of a large head rotated
        {"name": "rotary_train_part_fp16", "kind": "rotary_train", "b": 1, "s": 1531, "hq": 16,
         "hkv": 2, "d": 192, "rot": 64, "interleaved": True, "scaling": "linear", "far": 0,
         "dtype": "fp16"},
        # a decode step's layer: one token of each of 64 requests
        {"name": "append_decode_64", "kind": "append", "r": 64, "ctx_lo": 10, "ctx_hi": 4000,
         "new_lo": 1, "new_hi": 1, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "interleaved": False,
         "scaling": "wavelength", "block": 64, "dtype": "bf16"},
        # seven prompts in one step, ragged, small blocks, half of an odd head rotated
        {"name": "append_prompts_fp16", "kind": "append", "r": 7, "ctx_lo": 1, "ctx_hi": 500,
         "new_lo": 500, "new_hi": 6000, "hq": 16, "hkv": 8, "d": 80, "rot": 40,
         "interleaved": True, "scaling": "none", "block": 16, "dtype": "fp16"},
        # drafts to be verified, in fp32; their blocks are read as a 16-bit product takes them (in fp32
        # a code that lies on a border between two shows as a difference of the whole step)
        {"name": "append_drafts_fp32", "kind": "append", "r": 9, "ctx_lo": 0, "ctx_hi": 3000,
         "new_lo": 1, "new_hi": 5, "hq": 12, "hkv": 4, "d": 64, "rot": 64, "interleaved": False,
         "scaling": "linear", "block": 32, "dtype": "fp32"},
        # one user's answer from four beams, twice as many candidates as beams
        {"name": "beam_1x4_fp16", "kind": "beam", "g": 1, "k": 4, "v": 32000, "num": 8,
         "masked": 0.0, "done": 0.0, "first": False, "dtype": "fp16"},
        # constrained answers in fp32: most of an odd vocabulary masked, some beams at their end
        {"name": "beam_masked_9x5_fp32", "kind": "beam", "g": 9, "k": 5, "v": 50021, "num": 10,
         "masked": 0.9, "done": 0.2, "first": False, "dtype": "fp32"},
        # a full batch: 64 requests of 8 beams over a large vocabulary
        {"name": "beam_64x8", "kind": "beam", "g": 64, "k": 8, "v": 128256, "num": 16,
         "masked": 0.0, "done": 0.05, "first": False, "dtype": "bf16"},
        # four requests of four beams after a step, 8 layers' caches: latency
        {"name": "reorder_4x4", "kind": "reorder", "g": 4, "k": 4, "ctx_lo": 100, "ctx_hi": 2000,
         "gen": 150, "layers": 8, "hkv": 4, "d": 64, "block": 64, "gone": 0.0},
        # 64 requests of 8 beams, some of them at their end and given back
        {"name": "reorder_64x8", "kind": "reorder", "g": 64, "k": 8, "ctx_lo": 100, "ctx_hi": 2000,
         "gen": 200, "layers": 4, "hkv": 4, "d": 128, "block": 32, "gone": 0.05},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotary", "rotary_train", "append", "append", "beam", "beam", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("rotary", "rotary_train", "append"):
        d = rng.choice([64, 72, 80, 96, 100, 128, 128, 192, 256])
        case = {"kind": kind, "d": d, "rot": rng.choice([d, d, d // 4 * 2, 2 * rng.randint(1, d // 2)]),
                "interleaved": rng.random() < 0.4, "dtype": dtype,
                "scaling": rng.choice(["none", "linear", "base", "ramp", "wavelength", "list"]),
                "hkv": rng.choice([1, 2, 4, 5, 8, 8])}
        case["hq"] = case["hkv"] * rng.choice([1, 2, 4, 4, 7, 8])
        if kind != "append":
            case.update(b=rng.choice([1, 1, 2, 5]), s=log(1, 8192), far=rng.choice([0, 0, 4000000]))
            while case["b"] * case["s"] * (case["hq"] + case["hkv"]) * d * SIZE[dtype] > 8192 * 40 * 256:
                case["s"] = case["s"] // 2
            return case
        case.update(r=log(1, 64), ctx_lo=rng.choice([0, 1, 100]), ctx_hi=log(200, 16000),
                    block=rng.choice([16, 32, 64, 128]))
        # generation, drafts, or prompts
        case["new_lo"], case["new_hi"] = rng.choice([(1, 1), (1, rng.randint(2, 9)),
                                                     (rng.randint(20, 100), log(100, 2048))])
        while _tokens(case) * (case["hq"] + 2 * case["hkv"]) * d > 17000 * 16 * 128:
            case["r"] = max(1, case["r"] // 2)
            case["new_hi"] = max(case["new_lo"], case["new_hi"] * 3 // 4)
        return case
    if kind == "beam":
        k, v = rng.choice([1, 2, 3, 4, 5, 8, 16]), log(1000, 130000)
        g = log(1, 64)
        while g * k * v * SIZE[dtype] > 64 * 8 * 128256 * 2:
            g = max(1, g // 2)
        return {"kind": kind, "g": g, "k": k, "v": v, "num": rng.choice([k, 2 * k, min(64, 3 * k + 1)]),
                "masked": rng.choice([0.0, 0.0, 0.5]), "done": rng.choice([0.0, 0.2]),
                "first": rng.random() < 0.2, "dtype": dtype}
    case = {"kind": kind, "g": log(1, 64), "k": rng.choice([1, 2, 3, 4, 5, 8]), "ctx_lo": 1,
            "ctx_hi": log(50, 2000), "gen": rng.choice([0, log(1, 300)]), "layers": rng.randint(1, 9),
            "hkv": rng.choice([1, 2, 4]), "d": rng.choice([64, 80, 128]),
            "block": rng.choice([16, 32, 64, 128]), "gone": rng.choice([0.0, 0.1])}
    while sum(map(sum, _beam_lens(case))) * case["layers"] * case["hkv"] * case["d"] > 1e8:
        case["g"], case["layers"] = max(1, case["g"] // 2), max(1, case["layers"] // 2)
    return case


# ------------------------------------------------------------------ sizes of a case

def _lens(case):
    """(context, new tokens) of each request: ragged, of the case alone."""
    rng = random.Random(case["r"] * 1_000_003 + case["ctx_hi"] * 101 + case["new_hi"])
    lo, hi = max(1, case["ctx_lo"]), max(1, case["ctx_hi"])
    ctx = [int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) for _ in range(case["r"])]
    if case["ctx_lo"] == 0:
        ctx[0] = 0
    return ctx, [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["r"])]


def _tokens(case):
    return sum(_lens(case)[1])


def _beam_lens(case):
    """(prompt, answered tokens of all its beams) of each request, of the case alone."""
    rng = random.Random(case["g"] * 1_000_003 + case["ctx_hi"] * 101 + case["gen"])
    prompts = [int(round(math.exp(rng.uniform(math.log(case["ctx_lo"]), math.log(case["ctx_hi"])))))
               for _ in range(case["g"])]
    return prompts, [case["k"] * rng.randint(0, case["gen"]) for _ in range(case["g"])]


def _beam_rows(case):
    """Rows of blocks numbered from 0, lengths, parents: a tree of beams, of the case alone.

    Beams share a prompt's full blocks, and those of their answers that an ancestor filled; the last
    begun block is each one's own."""
    rng = random.Random(case["g"] * 7 + case["k"] * 131 + case["ctx_hi"] * 17 + case["gen"])
    b, k = case["block"], case["k"]
    rows, lens, parents, count = [], [], [], 0
    for prompt, answered in zip(*_beam_lens(case)):
        n = prompt + answered // k
        first = len(rows)
        mine = [[] for _ in range(k)]
        for j in range(-(-n // b)):
            whole = (j + 1) * b <= n
            if (j + 1) * b <= prompt:
                shared = 1
            elif whole:
                shared = max(1, k * (j + 1) * b // (2 * n))  # ancestors' blocks, ever fewer beams each
            else:
                shared = k
            for i in range(k):
                mine[i].append(count + i * shared // k)
            count += shared
        rows += mine
        lens += [n] * k
        if rng.random() < case["gone"]:
            parents += [-1] * k
        else:
            # better beams have more children
            parents += sorted(first + min(rng.randrange(k), rng.randrange(k)) for _ in range(k))
    return rows, lens, parents, count


def _copies(case):
    """Begun blocks that other children of a row need of their own."""
    _, lens, parents, _ = _beam_rows(case)
    seen, n = set(), 0
    for p in parents:
        if p >= 0:
            n += p in seen and lens[p] % case["block"] != 0
            seen.add(p)
    return n


def work(case):
    kind = case["kind"]
    if kind in ("rotary", "rotary_train"):
        n = case["b"] * case["s"] * (case["hq"] + case["hkv"])
        twice = 2 if kind == "rotary_train" else 1
        return {"bytes": twice * (2 * n * case["d"] * SIZE[case["dtype"]] + 4 * case["s"]),
                "flops": twice * 3 * n * case["rot"]}
    if kind == "append":
        ctx, new = _lens(case)
        b, hd = case["block"], case["hkv"] * case["d"]
        touched = sum(-(-(c + n) // b) - c // b for c, n in zip(ctx, new))
        held = sum(c + n - c // b * b for c, n in zip(ctx, new))
        size = SIZE[case["dtype"]]
        # queries in and out, new keys and values in, their codes out; codes of the touched blocks
        # in, values out
        return {"bytes": 2 * sum(new) * case["hq"] * case["d"] * size
                + 2 * hd * (sum(new) * (size + 1) + held + touched * b * 2)
                + touched * case["hkv"] * 16 + 12 * sum(new),
                "flops": 3 * sum(new) * (case["hq"] + case["hkv"]) * case["rot"]}
    if kind == "beam":
        rows = case["g"] * case["k"]
        return {"bytes": rows * (case["v"] * SIZE[case["dtype"]] + 5) + case["g"] * case["num"] * 20,
                "flops": 0}
    rows, lens, parents, count = _beam_rows(case)
    b, width = case["block"], max(map(len, rows)) + 2
    total = count + len(rows) + 3
    block = 2 * case["hkv"] * b * (-(-case["d"] // 64) * 64) + case["hkv"] * 8
    # used entries in, tables out, the stack in and out, lengths and parents; copied blocks
    return {"bytes": sum(map(len, rows)) * 4 + len(parents) * (width * 4 + 24) + total * 8
            + 2 * _copies(case) * block * case["layers"], "flops": 0}


# ------------------------------------------------------------------ inputs

def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (salt + 1) + seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


BASE, TRAINED = 10000.0, 4096.0


def _scaling(case):
    """What a checkpoint's configuration says of its frequencies."""
    return {"none": None, "linear": {"kind": "linear", "factor": 4.0},
            "base": {"kind": "base", "factor": 8.0},
            "ramp": {"kind": "ramp", "factor": 16.0, "length": TRAINED},
            "wavelength": {"kind": "wavelength", "factor": 8.0, "length": TRAINED},
            "list": {"kind": "list", "factors": [1.0 + 0.37 * i for i in range(case["rot"] // 2)],
                     "gain": 1.19}}[case["scaling"]]


def _frequencies(case):
    """(radians per position of each pair, float64; the rotated part's gain)."""
    rot, kind = case["rot"], case["scaling"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    base = BASE * 8.0 ** (rot / (rot - 2)) if kind == "base" and rot > 2 else BASE
    f = base ** (-2 * i / rot)
    if kind == "linear":
        return f / 4, 1.0
    if kind == "ramp":
        # pairs that turn over 32 times in the trained length keep their frequency, those that turn
        # less than once are scaled
        at = [rot * math.log(TRAINED / (2 * math.pi * n)) / (2 * math.log(BASE)) for n in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        share = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / 16 * share + f * (1 - share), 0.1 * math.log(16.0) + 1
    if kind == "wavelength":
        turns = TRAINED * f / (2 * math.pi)
        t = ((turns - 1) / 3).clamp(0, 1)
        return (1 - t) * f / 8 + t * f, 1.0
    if kind == "list":
        return f / (1 + 0.37 * i), 1.19
    return f, 1.0


def _rotation(state, case):
    """The frequencies, or the framework's handle of them."""
    if own:
        state["rotation"] = _package().rotary.rotation(
            case["rot"], BASE, scaling=_scaling(case), interleaved=case["interleaved"], device=DEV)
    else:
        state["f"], state["gain"] = _frequencies(case)


def _heads(case, tokens, g):
    """Queries and keys as parts of one product's output, some channels large."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = torch.randn(*tokens, hq + 2 * hkv, d, generator=g, device=DEV)
    x *= 1 + 3 * (torch.arange(d, device=DEV) % 17 == 5).float()
    x = x.to(DTYPES[case["dtype"]])
    return x[..., :hq, :], x[..., hq:hq + hkv, :], x[..., hq + hkv:, :]


def prepare(case, seed):
    kind = case["kind"]
    state = {"case": case}
    if kind in ("rotary", "rotary_train"):
        g = _gen(seed)
        b, s = case["b"], case["s"]
        q, k, _ = _heads(case, (b, s), g)
        if case["far"]:
            positions = torch.randint(case["far"] // 2, case["far"], (b, s), generator=g, device=DEV)
        else:
            positions = torch.arange(s, device=DEV).expand(b, s)
        state.update(q=q, k=k, positions=positions.to(torch.int32) if kind == "rotary" else positions)
        if kind == "rotary_train":
            state.update(q=q.detach().requires_grad_(True), k=k.detach().requires_grad_(True),
                         gq=torch.randn(q.shape, generator=g, device=DEV).to(q.dtype),
                         gk=torch.randn(k.shape, generator=g, device=DEV).to(q.dtype))
        _rotation(state, case)
        return state
    if kind == "beam":
        g = _gen(seed, 1)
        n, k, v = case["g"], case["k"], case["v"]
        # logits of a model: a broad spread with a few likely tokens in each row
        x = torch.randn(n * k, v, generator=g, device=DEV).mul_(2.0)
        likely = torch.randint(0, v, (n * k, 10), generator=g, device=DEV)
        x.scatter_add_(1, likely, torch.rand(n * k, 10, generator=g, device=DEV) * 12)
        if case["masked"]:
            x.masked_fill_(torch.rand(n * k, v, generator=g, device=DEV) < case["masked"], -math.inf)
        # log probabilities of the answers so far
        scores = torch.rand(n, k, generator=g, device=DEV).mul_(-9).sub_(20).sort(1, descending=True)[0]
        if case["first"]:
            scores[:, 0], scores[:, 1:] = 0, -math.inf
        done = torch.rand(n, k, generator=g, device=DEV) < case["done"]
        state.update(x=x.to(DTYPES[case["dtype"]]).view(n, k, v), scores=scores, done=done)
        return state
    if kind == "reorder":
        rows, lens, parents, count = _beam_rows(case)
        g = _gen(seed, 2)
        total = count + len(rows) + 3
        perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
        tables = torch.full((len(rows), max(map(len, rows)) + 2), -1, dtype=torch.int32)
        for i, row in enumerate(rows):
            tables[i, :len(row)] = perm[row]
        free = torch.full((total,), -1, dtype=torch.int32)
        free[:total - count] = perm[count:].to(torch.int32)
        shape = (total, case["hkv"], case["block"], -(-case["d"] // 64) * 64)
        caches = []
        for _ in range(case["layers"]):
            codes = [torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
                     for _ in range(2)]
            scales = torch.rand(total, case["hkv"], 2, generator=g, device=DEV).mul_(0.03)
            caches.append((*codes, scales))
        state.update(tables=tables.to(DEV), lens=_i32(lens), free=free.to(DEV),
                     num_free=_i32([total - count]), total=total, caches=caches,
                     parents=torch.tensor(parents, dtype=torch.int64, device=DEV))
        return state

    ctx, new = _lens(case)
    g = _gen(seed, 3)
    b, h, d = case["block"], case["hkv"], case["d"]
    dp = -(-d // 64) * 64
    need = [-(-(c + n) // b) for c, n in zip(ctx, new)]
    perm = torch.randperm(sum(need) + 5, generator=torch.Generator().manual_seed(seed))
    tab, at = torch.full((case["r"], max(need)), -1, dtype=torch.int64), 0
    for r, n in enumerate(need):
        tab[r, :n] = perm[at:at + n]
        at += n
    shape = (len(perm), h, b, dp)
    for name in ("k_codes", "v_codes"):
        codes = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
        state[name] = codes.mul_(35).round_().clamp_(-127, 127).to(torch.int8)
        del codes
    # a block's scale: its largest value over 127, about 3.5 deviations, more in some blocks
    state["scales"] = (3.6 / 127) * torch.exp(0.25 * torch.randn(len(perm), h, 2, generator=g,
                                                                 device=DEV))
    state["q"], state["k"], state["v"] = _heads(case, (sum(new),), g)
    req = torch.repeat_interleave(torch.arange(case["r"]), torch.tensor(new))
    starts = torch.tensor([0] + new).cumsum(0)
    pos = torch.arange(sum(new)) - starts[req] + torch.tensor(ctx)[req]
    state["slots"] = (tab[req, pos // b] * b + pos % b).to(DEV)
    state["positions"] = pos.to(torch.int32).to(DEV)
    state["blocks"] = torch.cat([tab[r, c // b:-(-(c + n) // b)]
                                 for r, (c, n) in enumerate(zip(ctx, new))]).to(torch.int32).to(DEV)
    _rotation(state, case)
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


def _read_as(case):
    return torch.bfloat16 if case["dtype"] == "fp32" else DTYPES[case["dtype"]]


def _angles(s):
    a = s["positions"].double()[..., None] * s["f"]
    return (a.cos() * s["gain"]).float()[..., None, :], (a.sin() * s["gain"]).float()[..., None, :]


def _plain_rotate(x, cos, sin, case):
    """The rotated heads in fp32."""
    rot, x = case["rot"], x.float()
    if case["interleaved"]:
        lo, hi = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([lo * cos - hi * sin, hi * cos + lo * sin], -1).flatten(-2)
    else:
        lo, hi = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rotary(s):
    case = s["case"]
    with torch.no_grad():
        cos, sin = _angles(s)
        out = {"q": _plain_rotate(s["q"], cos, sin, case).to(s["q"].dtype),
               "k": _plain_rotate(s["k"], cos, sin, case).to(s["q"].dtype)}
        if case["kind"] == "rotary_train":
            out.update(dq=_plain_rotate(s["gq"], cos, -sin, case).to(s["q"].dtype),
                       dk=_plain_rotate(s["gk"], cos, -sin, case).to(s["q"].dtype))
    return out


def _plain_append(s):
    case, slots, scales = s["case"], s["slots"], s["scales"]
    b, d, dt = case["block"], case["d"], _read_as(case)
    cos, sin = _angles(s)
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
    for i, (x, codes, out_of, into) in enumerate((
            (_plain_rotate(s["k"], cos, sin, case), s["k_codes"], _k_out, _k_in),
            (s["v"].float(), s["v_codes"], _v_out, _v_in))):
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
    q = _plain_rotate(s["q"], cos, sin, case).to(s["q"].dtype)
    return {"q": q, "k": out[0], "v": out[1], "scales": scales[touched]}


def _plain_beam(s):
    case, x, scores = s["case"], s["x"].double(), s["scores"].double()
    n, k, v = x.shape
    # in 64 bits: candidates of different beams may lie as close as the rounding of 32-bit sums
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    value = x - lse + scores[..., None]
    ended = torch.full((v,), -math.inf, device=DEV, dtype=torch.float64)
    ended[PAD] = 0
    value = torch.where(s["done"][..., None], ended + scores[..., None], value).view(n, k * v)
    # equal ones in the order of beams and tokens
    best, order = torch.sort(value, dim=-1, descending=True, stable=True)
    best, order = best[:, :case["num"]], order[:, :case["num"]]
    rows = torch.arange(n, device=DEV)[:, None] * k + order // v
    return {"scores": best.float(), "parents": rows, "tokens": order % v}


def _plain_reorder(s):
    b, tables, parents = s["case"]["block"], s["tables"], s["parents"]
    r, w = tables.shape
    n, total = parents.numel(), s["total"]
    used = ((s["lens"] + b - 1) // b).clamp(max=w)
    col, child = torch.arange(w, device=DEV), torch.arange(n, device=DEV)
    old = torch.where(col < used[:, None], tables, -1)
    kept, at = parents >= 0, parents.clamp(min=0)
    first = torch.full((r,), n, device=DEV)
    first = first.scatter_reduce(0, at, torch.where(kept, child, n), "amin")
    now = torch.where(kept[:, None], old[at], -1)
    lens = torch.where(kept, s["lens"][at], 0)
    # blocks of the old rows, and those that a new row holds
    marks = []
    for t in (old, now):
        held = torch.zeros(total + 1, dtype=torch.bool, device=DEV)
        held[torch.where(t >= 0, t, total).view(-1).long()] = True
        marks.append(held[:total])
    freed = marks[0] & ~marks[1]
    place = torch.where(freed, s["num_free"] + torch.cumsum(freed, 0) - 1, total)
    index = torch.arange(total + 1, device=DEV, dtype=torch.int32)
    stack = torch.full((total + 1,), -1, dtype=torch.int32, device=DEV)
    stack[:total] = torch.where(index[:total] < s["num_free"], s["free"], -1)
    stack[place] = index[:total]
    top = s["num_free"] + freed.sum()
    # children after the first one need a begun block of their own
    last = (lens // b).clamp(max=w - 1).long()[:, None]
    begun = now.gather(1, last)[:, 0]
    copy = kept & (lens % b > 0) & (first[at] != child) & (begun >= 0)
    take = top - torch.cumsum(copy, 0)
    fresh = torch.where(take >= 0, stack[take.clamp(min=0)], -1)
    sources, targets = torch.where(copy, begun, -1), torch.where(copy, fresh, -1)
    now.scatter_(1, last, torch.where(copy, fresh, begun)[:, None])
    left = top - copy.sum()
    stack = torch.where(index[:total] < left, stack[:total], -1)
    moves = targets >= 0
    src, dst = sources[moves].long(), targets[moves].long()
    for cache in s["caches"]:
        for t in cache:
            t[dst] = t[src]
    return {"tables": now, "lens": lens, "free": stack, "num_free": left.to(torch.int32),
            "sources": sources, "targets": targets, "caches": s["caches"]}


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"rotary": _plain_rotary, "rotary_train": _plain_rotary, "append": _plain_append,
                "beam": _plain_beam, "reorder": _plain_reorder}[kind](s)
    amd = _package()
    if kind in ("rotary", "rotary_train"):
        q, k = amd.rotary.rotate_qk(s["q"], s["k"], s["positions"], s["rotation"])
        if kind == "rotary":
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["gq"], s["gk"]])
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if kind == "append":
        q = amd.kv8.rotate_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotation"],
                                  s["k_codes"], s["v_codes"], s["scales"])
        k, v, scales = amd.kv8.read(s["k_codes"], s["v_codes"], s["scales"], s["blocks"],
                                    case["d"], _read_as(case))
        return {"q": q, "k": k, "v": v, "scales": scales}
    if kind == "beam":
        best = amd.beam_select(s["x"], s["scores"], case["num"], finished=s["done"], pad_id=PAD)
        return {"scores": best.scores, "parents": best.parents, "tokens": best.tokens}
    step = amd.kv8.reorder(s["parents"], s["lens"], s["tables"], s["free"], s["num_free"],
                           case["block"], s["total"])
    amd.kv8.copy_blocks(s["caches"], step.sources, step.targets)
    return {"tables": step.block_tables, "lens": step.seq_lens, "free": step.free_blocks,
            "num_free": step.num_free, "sources": step.sources, "targets": step.targets,
            "caches": s["caches"]}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    kind = case["kind"]
    if kind == "reorder":
        return None  # whole numbers and copies only
    s = prepare(case, seed)
    if kind == "beam":
        n, k, v = s["x"].shape
        out = {"scores": [], "parents": [], "tokens": []}
        for g in range(n):
            value = torch.log_softmax(s["x"][g].double(), -1) + s["scores"][g].double()[:, None]
            for i in range(k):
                if s["done"][g, i]:
                    value[i] = -math.inf
                    value[i, PAD] = s["scores"][g, i].double()
            value = value.view(-1)
            least = torch.topk(value, case["num"])[0][-1]
            place = torch.nonzero(value >= least)[:, 0]
            if least == -math.inf:  # any of the impossible ones, the first first
                place = torch.cat([torch.nonzero(value > least)[:, 0],
                                   torch.nonzero(value == least)[:case["num"], 0]])
            pairs = sorted(zip((-value[place]).tolist(), place.tolist()))[:case["num"]]
            out["scores"].append([-a for a, _ in pairs])
            out["parents"].append([g * k + j // v for _, j in pairs])
            out["tokens"].append([j % v for _, j in pairs])
        return {"scores": torch.tensor(out["scores"], dtype=torch.float64, device=DEV),
                "parents": torch.tensor(out["parents"], device=DEV),
                "tokens": torch.tensor(out["tokens"], device=DEV)}

    f, gain = _frequencies(case)
    turn = torch.polar(torch.full_like(f, gain).expand(*s["positions"].shape, -1).contiguous(),
                       s["positions"].double()[..., None] * f)[..., None, :]

    def rotated(x, turn):
        rot, y = case["rot"], x.detach().double().clone()
        places = torch.arange(rot, device=DEV)
        lo, hi = (places[0::2], places[1::2]) if case["interleaved"] else places.chunk(2)
        z = torch.complex(y[..., lo], y[..., hi]) * turn
        y[..., lo], y[..., hi] = z.real, z.imag
        return y

    q = rotated(s["q"], turn)
    if kind == "rotary":
        return {"q": q, "k": rotated(s["k"], turn)}
    if kind == "rotary_train":
        return {"q": q, "k": rotated(s["k"], turn), "dq": rotated(s["gq"], turn.conj()),
                "dk": rotated(s["gk"], turn.conj())}
    b, d, n = case["block"], case["d"], s["blocks"].numel()
    where = {int(k): i for i, k in enumerate(s["blocks"].tolist())}
    slots = s["slots"].cpu()
    run_of = torch.tensor([where[int(x)] for x in (slots // b).tolist()], device=DEV)
    off = (slots % b).to(DEV)
    out, new_scales = [], []
    for i, (name, x) in enumerate((("k", rotated(s["k"], turn)), ("v", s["v"].double()))):
        raw = s[name + "_codes"][s["blocks"].long()]
        dp = raw.shape[-1]
        tok = torch.arange(b, device=DEV)[:, None]
        dd = torch.arange(dp, device=DEV)[None, :]
        if name == "k":
            at = (tok // 16 * dp * 16 + dd // 64 * 1024 + tok % 16 // 4 * 256
                  + dd % 64 // 16 * 64 + tok % 4 * 16 + dd % 16)
        else:
            at = tok // 16 * dp * 16 + dd * 16 + tok % 16
        values = raw.reshape(n, -1, b * dp)[:, :, at].double()
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
    return {"q": q, "k": out[0], "v": out[1], "scales": torch.stack(new_scales, -1)}
