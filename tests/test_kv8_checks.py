"""What the cache's operators and token_logprobs refuse, before anything is launched: the ops'
bodies on CPU tensors with a library that records its calls, and the C ABI itself."""

import contextlib
import ctypes

import pytest
import torch

from ojasx_amd import _native as N
from ojasx_amd import kv8, serve_ops as S


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name) or 0


@pytest.fixture
def library(monkeypatch):
    fake = _Library()
    monkeypatch.setattr(N, "lib", lambda: fake)
    monkeypatch.setattr(N, "require_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(N, "stream_handle", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return fake


def _cache(blocks=4, heads=2, block=16, d=80):
    return kv8.KV8Cache(blocks, heads, d, block, device="cpu")


I32 = torch.int32


def _plan(**change):
    a = dict(seq_lens=torch.zeros(3, dtype=I32), new_lens=torch.ones(3, dtype=I32),
             block_tables=torch.zeros(3, 5, dtype=I32), free_blocks=torch.arange(4, dtype=I32),
             num_free=torch.tensor([4], dtype=I32), block_size=16, num_tokens=3)
    a.update(change)
    return S.kv8_plan(*a.values())


def test_plan_is_taken_and_refused(library):
    out = _plan()
    assert library.calls == ["ojx_kv8_plan"]
    assert [t.shape[0] for t in out] == [3, 3, 3, 4, 3, 1] and out[0].dtype == torch.int64
    for change in (dict(new_lens=torch.ones(2, dtype=I32)), dict(seq_lens=torch.zeros(3)),
                   dict(block_tables=torch.zeros(2, 5, dtype=I32)),
                   dict(block_tables=torch.zeros(3, 5, dtype=torch.int64)),
                   dict(block_tables=torch.zeros(5, 3, dtype=I32).t()),
                   dict(num_free=torch.zeros(2, dtype=I32)), dict(block_size=48),
                   dict(free_blocks=torch.arange(4)), dict(num_tokens=-1)):
        with pytest.raises(RuntimeError):
            _plan(**change)
    assert len(library.calls) == 1


def test_append_is_taken_and_refused(library):
    c = _cache()
    k = torch.zeros(5, 2, 80, dtype=torch.bfloat16)
    slots = torch.zeros(5, dtype=torch.int64)
    c.append(k, k, slots)
    assert library.calls == ["ojx_kv8_append"]
    for args in ((k, k.float(), slots), (k, k[:, :1], slots), (k[0], k[0], slots),
                 (k, k, slots.int()), (k, k, slots[:4]), (k[:, :, :60], k[:, :, :60], slots),
                 (k.double(), k.double(), slots), (k[:, :1], k[:, :1], slots)):
        with pytest.raises(RuntimeError):
            c.append(*args)
    for codes in (c.k_codes.float(), c.k_codes[:, :, ::2], c.k_codes[0], c.k_codes[:3]):
        with pytest.raises(RuntimeError):
            kv8.append(k, k, slots, codes, c.v_codes, c.scales)
    for scales in (c.scales.half(), c.scales[:3], c.scales[..., 0]):
        with pytest.raises(RuntimeError):
            kv8.append(k, k, slots, c.k_codes, c.v_codes, scales)
    assert len(library.calls) == 1


def test_read_and_attention_are_taken_and_refused(library):
    c = _cache()
    blocks = torch.zeros(3, dtype=I32)
    k, v, s = c.read(blocks)
    assert k.shape == v.shape == (3, 16, 2, 80) and s.shape == (3, 2, 2)
    for args in ((blocks.long(), torch.float16), (blocks, torch.float64)):
        with pytest.raises(RuntimeError):
            c.read(*args)
    with pytest.raises(RuntimeError):
        kv8.read(c.k_codes, c.v_codes, c.scales, blocks, 129, torch.float16)
    q = torch.zeros(3, 6, 80, dtype=torch.float16)
    tables, lens = torch.zeros(3, 2, dtype=I32), torch.ones(3, dtype=I32)
    calls = len(library.calls)
    out, lse = c.attention(q, tables, lens, return_lse=True)
    assert out.shape == q.shape and lse.shape == (3, 6)
    assert library.calls[calls:] == ["ojx_kv8_attention_workspace_bytes", "ojx_kv8_attention"]
    for args in ((q[0], tables, lens), (q.double(), tables, lens), (q[..., :20], tables, lens),
                 (q, tables.long(), lens), (q, tables[:2], lens), (q, tables, lens.long()),
                 (q, tables, lens, torch.zeros(3, dtype=I32)),
                 (q, tables, lens, torch.zeros(4))):
        with pytest.raises(RuntimeError):
            c.attention(*args)


def test_a_cache_that_cannot_be():
    for args in ((4, 2, 80, 48), (4, 2, 0, 16), (4, 2, 257, 16), (4, 0, 64, 16), (-1, 2, 64, 16)):
        with pytest.raises(RuntimeError):
            kv8.KV8Cache(*args, device="cpu")


def test_token_logprobs_is_taken_and_refused(library):
    x, ids = torch.zeros(2, 3, 50), torch.zeros(2, 3, dtype=torch.int64)
    out = S.token_logprobs(x, ids, 4)
    assert [tuple(t.shape) for t in out] == [(2, 3)] * 3 + [(2, 3, 4)] * 2 + [(2, 3, 2)]
    for args in ((x, ids.int(), 4), (x, ids[0], 4), (x, ids, 51), (x, ids, -1), (x.double(), ids, 4),
                 (x[..., :0], ids, 0), (torch.zeros(2, 100), ids[0, :2], 65)):
        with pytest.raises(RuntimeError):
            S.token_logprobs(*args)
    f = torch.zeros(2, 3)
    S.token_logprobs_bwd(x, ids, f, out[5], out[4], f, None, None, out[3])
    for change in (dict(h=f.double()), dict(stats=f), dict(top=out[4].int()), dict(top=out[4][0]),
                   dict(g=f.half()), dict(gt=f)):
        a = dict(h=f, stats=out[5], top=out[4], g=f, gt=out[3])
        a.update(change)
        with pytest.raises(RuntimeError):
            S.token_logprobs_bwd(x, ids, a["h"], a["stats"], a["top"], a["g"], None, None, a["gt"])


def test_cpu_tensors_raise():
    c = _cache()
    with pytest.raises(RuntimeError, match="ROCm"):
        c.attention(torch.zeros(1, 2, 80), torch.zeros(1, 1, dtype=I32), torch.ones(1, dtype=I32))


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = N.lib()
    P = ctypes.c_void_p(256)  # never read: every call is refused or has nothing to do
    n = ctypes.c_size_t(7)
    plan = [P, P, 1, P, 4, 4, P, 4, P, 16, 1, P, P, P, P, P, P, None]

    def bad(fn, args, i, value, code):
        a = list(args)
        a[i] = value
        assert fn(*a) == code, (fn, i, value)

    for i, value, code in ((2, -1, -1), (9, 24, -2), (10, -1, -1), (10, 1 << 31, -1), (8, None, -1),
                           (0, None, -1), (11, None, -1), (5, -1, -1)):
        bad(lib.ojx_kv8_plan, plan, i, value, code)
    bad(lib.ojx_kv8_plan, [P, P, 2, P, 3, 4, P, 4, P, 16, 1, P, P, P, P, P, P, None], 0, P, -1)
    app = [P, P, P, 4, 2, 16, 80, P, 160, 80, P, 160, 80, 2, P, 3, None]
    for i, value, code in ((3, -1, -1), (4, 0, -1), (5, 20, -2), (6, 0, -2), (6, 257, -2), (13, 3, -3),
                           (15, -1, -1), (7, None, -1), (8, -1, -1), (0, None, -1),
                           (0, ctypes.c_void_p(8), -2)):
        bad(lib.ojx_kv8_append, app, i, value, code)
    bad(lib.ojx_kv8_append, app, 15, 0, 0)
    read = [P, P, P, 4, 2, 16, 80, P, 3, 2, P, P, P, None]
    for i, value, code in ((9, 5, -3), (8, -2, -1), (10, ctypes.c_void_p(8), -2), (12, None, -1)):
        bad(lib.ojx_kv8_read, read, i, value, code)
    bad(lib.ojx_kv8_read, read, 8, 0, 0)
    att = [P, 480, 80, 3, 6, 2, P, P, P, 4, 2, 16, 80, P, 2, 2, P, P, 3, 1, 32, 0.1, 0, P, None,
           None, 0, None]
    for i, value, code in ((4, 5, -1), (4, 0, -1), (5, 9, -3), (12, 300, -2), (18, -1, -1),
                           (21, float("nan"), -1), (21, float("inf"), -1), (22, -1, -1),
                           (26, 16, -1), (25, ctypes.c_void_p(8), -2), (1, -1, -1), (0, None, -1),
                           (14, 1, -1), (3, 1 << 31, -1)):
        bad(lib.ojx_kv8_attention, att, i, value, code)
    no_starts = list(att)
    no_starts[17], no_starts[18] = None, 2
    assert lib.ojx_kv8_attention(*no_starts) == -1
    no_tokens = list(att)
    no_tokens[3] = 0
    assert lib.ojx_kv8_attention(*no_tokens) == 0
    assert lib.ojx_kv8_attention_workspace_bytes(3, 3, 6, 2, 80, 0, 1, 32, 9, ctypes.byref(n)) == -3
    assert lib.ojx_kv8_attention_workspace_bytes(3, 3, 6, 2, 80, 0, 1, 32, 2, None) == -1
    assert lib.ojx_kv8_attention_workspace_bytes(0, 0, 6, 2, 80, 0, 1, 32, 2, ctypes.byref(n)) == 0
    assert n.value == 0
    lp = [P, 100, 3, 100, 0, P, 5, P, P, P, P, P, P, None, 0, None]
    for i, value, code in ((1, 99, -1), (3, 0, -1), (4, 7, -3), (6, 65, -1), (6, -1, -1), (0, None, -1),
                           (10, None, -1), (14, 8, -1)):
        bad(lib.ojx_token_logprobs, lp, i, value, code)
    bad(lib.ojx_token_logprobs, lp, 2, 0, 0)
    back = [P, 100, 3, 100, 0, P, P, P, 5, P, P, P, P, P, P, None]
    for i, value, code in ((3, -4, -1), (4, 7, -3), (9, None, -1), (14, None, -1), (6, None, -1)):
        bad(lib.ojx_token_logprobs_bwd, back, i, value, code)
    bad(lib.ojx_token_logprobs_bwd, back, 2, 0, 0)
