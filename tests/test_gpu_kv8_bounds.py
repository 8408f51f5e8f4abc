"""Attention under bounds, windows and workspaces that do not fit the batch."""

import ctypes

import numpy as np
import pytest
import torch

import kv8_plain as P
from ojasx_amd import _native as N
from test_gpu_kv8 import DEV, DTYPES, _batch, _check_attention, _i32, _make

pytestmark = pytest.mark.gpu


def _code(dtype):
    return N.DTYPE_CODE[dtype]


def _workspace_bytes(q, cache, requests, window, max_query, max_seq):
    n = ctypes.c_size_t(0)
    t, heads, d = q.shape
    N.check(N.lib().ojx_kv8_attention_workspace_bytes(
        t, requests, heads, cache.k_codes.shape[1], d, window, max_query, max_seq, _code(q.dtype),
        ctypes.byref(n)), "workspace")
    return n.value


def _call(cache, q, tables, lens, starts, max_query, max_seq, scale, window=0, ws=None, ws_bytes=0):
    """The C entry point on outputs that held NaN."""
    t, heads, d = q.shape
    out = torch.full_like(q, float("nan"), memory_format=torch.contiguous_format)
    lse = torch.full((t, heads), float("nan"), device=DEV)
    blocks, kv_heads, block, _ = cache.k_codes.shape
    N.check(N.lib().ojx_kv8_attention(
        N.ptr(q), q.stride(0), q.stride(1), t, heads, _code(q.dtype), N.ptr(cache.k_codes),
        N.ptr(cache.v_codes), N.ptr(cache.scales), blocks, kv_heads, block, d, N.ptr(tables),
        tables.stride(0), tables.shape[1], N.ptr(lens), N.ptr(starts), lens.numel(), max_query,
        max_seq, scale, window, N.ptr(out), N.ptr(lse), N.ptr(ws), ws_bytes,
        N.stream_handle(DEV)), "attention")
    return out, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,group", [(64, 4), (100, 1), (256, 2)])
@pytest.mark.parametrize("most", [0, 1, 3, 17, 64, 89])
def test_rows_past_the_longest_query_are_zero(dtype, d, group, most):
    new = [5, 1, 90, 0, 70, 2]
    tables, lens, starts, total = _batch([30, 0, 9, 4, 200, 1], new, 16)
    cache = _make(16, 2, d, total)
    q = torch.randn(starts[-1], 2 * group, d).to(dtype).to(DEV)
    full, full_lse = _call(cache, q, _i32(tables), _i32(lens), _i32(starts), 90, max(lens), 0.1)
    ws_bytes = _workspace_bytes(q, cache, 6, 0, most, max(lens))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=DEV)
    for space in ((None, 0), (ws, ws_bytes)):
        out, lse = _call(cache, q, _i32(tables), _i32(lens), _i32(starts), most, max(lens), 0.1, 0,
                         *space)
        for a, b in zip(starts, starts[1:]):
            cut = min(b, a + most)
            # what is computed agrees with the call of the right bound (to the forms' roundings)
            torch.testing.assert_close(out[a:cut], full[a:cut], rtol=2e-2, atol=2e-2)
            torch.testing.assert_close(lse[a:cut], full_lse[a:cut], rtol=1e-3, atol=1e-3)
            assert not out[cut:b].any() and torch.isneginf(lse[cut:b]).all()
    assert torch.isfinite(full).all() and not full_lse.isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 2, 1], [40, 1, 70]])
def test_tokens_before_the_first_request_are_zero(dtype, new):
    tables, lens, starts, total = _batch([30, 0, 9], new, 16)
    cache = _make(16, 2, 64, total)
    q = torch.randn(starts[-1] + 7, 4, 64).to(dtype).to(DEV)
    t, n = _i32(tables), _i32(lens)
    want, want_lse = _call(cache, q[7:], t, n, _i32(starts), max(new), max(lens), 0.1)
    out, lse = _call(cache, q, t, n, _i32([s + 7 for s in starts]), max(new), max(lens), 0.1)
    assert not out[:7].any() and torch.isneginf(lse[:7]).all()
    assert torch.equal(out[7:], want) and torch.equal(lse[7:], want_lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 2, 1], [40, 1, 70]])
def test_rows_outside_q_are_left_out(dtype, new):
    # the last request's rows go on past q: those that q holds are computed
    tables, lens, starts, total = _batch([30, 0, 9], new, 16)
    cache = _make(16, 2, 64, total)
    q = torch.randn(starts[-1] + 5, 4, 64).to(dtype).to(DEV)
    t, n = _i32(tables), _i32([*lens[:2], lens[2] + 5])
    s = _i32([*starts[:3], starts[3] + 5])
    want, want_lse = _call(cache, q, t, n, s, max(new) + 5, max(lens) + 5, 0.1)
    out, lse = _call(cache, q[:starts[3]], t, n, s, max(new) + 5, max(lens) + 5, 0.1)
    assert torch.equal(out, want[:starts[3]]) and torch.equal(lse, want_lse[:starts[3]])
    assert not lse.isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [33, 64, 65, 70, 100, 150, 2 ** 31 - 1, 2 ** 40])
def test_windows_longer_than_what_the_table_holds(dtype, window):
    # requests of more tokens than their four blocks of 16: the window ends where it does
    tables, _, starts, total = _batch([60, 60, 60], [4, 4, 4], 16)
    tables = [row[:4] for row in tables]
    cache = _make(16, 1, 64, total)
    for new in ([1, 1, 1], [1, 4, 30]):
        starts = [0, *np.cumsum(new).tolist()]
        q = torch.randn(starts[-1], 2, 64).to(dtype).to(DEV)
        _check_attention(cache, q, tables, [64, 100, 120], starts, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1] * 3, [9, 3, 1], [70, 5, 130]])
def test_a_smaller_workspace_lowers_the_split(dtype, new):
    tables, lens, starts, total = _batch([3000, 2500, 17], new, 64)
    cache = _make(64, 2, 128, total)
    q = torch.randn(starts[-1], 4, 128).to(dtype).to(DEV)
    t, n = _i32(tables), _i32(lens)
    s = None if max(new) == 1 else _i32(starts)
    need = _workspace_bytes(q, cache, 3, 0, max(new), max(lens))
    assert need > 0
    k, v = P.codes_of(cache)
    sc = cache.scales.cpu().numpy()
    want = P.attention(q.float().cpu().numpy(), k, v, sc[:, :, 0], sc[:, :, 1], tables, lens,
                       starts, 0.1, 0, 64)[0]
    for share in (0.9, 0.5):
        size = int(need * share) // 16 * 16
        ws = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        out, lse = _call(cache, q, t, n, s, max(new), max(lens), 0.1, 0, ws, size)
        assert (ws[:size] != 0xA5).any()     # it is used
        assert (ws[size:] == 0xA5).all()
        # 127 scales of 0.02 e^1.5 at most and rounding to bf16 and 16-bit fixed point: under 0.1
        assert np.abs(out.double().cpu().numpy() - want).max() < 0.1 and not lse.isnan().any()


def test_a_longest_sequence_beyond_the_table_does_not_undo_the_split():
    """One token over 16128 keys.  Bounds longer than the table ask for other splits than the
    table's; what the workspace of one holds must not leave the other uncut: one workgroup would
    go through all 252 tiles of a key head, some 60 times the work of a part."""
    tables, lens, _, total = _batch([16127], [1], 64)
    cache = _make(64, 1, 128, total)
    q = torch.randn(1, 4, 128, dtype=torch.bfloat16, device=DEV)
    t, n = _i32(tables), _i32(lens)
    times = {}
    for bound in (16128, 131072):
        def call():
            return cache.attention(q, t, n, max_seq_len=bound)
        call()
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        best = float("inf")
        for _ in range(5):
            a.record()
            for _ in range(20):
                call()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times[bound] = best
    # parts of at most twice as many tiles: twice the time would be a lot
    assert times[131072] < 2 * times[16128], times
