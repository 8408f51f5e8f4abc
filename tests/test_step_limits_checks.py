"""Sizes past what a launch holds (2^32 threads in a dimension) are refused by the operators of a step's
positions and beams at the C ABI, before anything is launched."""

import ctypes

import pytest

from ojasx_amd import _native as N

P = ctypes.c_void_p(256)  # never read: every call is refused


@pytest.mark.parametrize("groups,beams", [(1 << 24, 1), (1 << 23, 1), (1 << 22, 2), (1 << 17, 64),
                                          ((1 << 30) // 64, 64)])
def test_beams(groups, beams):
    lib, n = N.lib(), ctypes.c_size_t(7)
    size = lib.ojx_beam_select_workspace_bytes
    assert size(groups, beams, 10, 1, 2, ctypes.byref(n)) == -1 and n.value == 0
    assert lib.ojx_beam_select(P, 10, groups, beams, 10, 2, P, None, 0, 1, P, P, P, P, 1 << 40, None) == -1
    # the most that there may be
    assert size(((1 << 23) - 1) // beams, beams, 10, 1, 2, ctypes.byref(n)) == 0 and n.value > 0


@pytest.mark.parametrize("rows,children", [(1, 1 << 26), (1, (1 << 25) + 1), ((1 << 25) + 1, 1), (1 << 30, 1)])
def test_reordered_rows(rows, children):
    lib, n = N.lib(), ctypes.c_size_t(7)
    size = lib.ojx_kv8_reorder_workspace_bytes
    assert size(rows, children, 4, 16, 9, ctypes.byref(n)) == -1 and n.value == 0
    assert lib.ojx_kv8_reorder(P, children, P, rows, P, 4, 4, P, 5, P, 16, 9, *[P] * 7, 1 << 40, None) == -1
    assert size(min(rows, 1 << 25), min(children, 1 << 25), 4, 16, 9, ctypes.byref(n)) == 0


def _heads(heads, d, at=256):
    return N.RotaryRows(x=at, y=at, x_batch=0, x_token=heads * d, x_head=d, y_batch=0, y_token=heads * d,
                        y_head=d, heads=heads)


@pytest.mark.parametrize("dtype,d,pairs,heads,tokens", [
    (2, 64, 32, 2, 1 << 30),    # 16 bytes of two heads by two a thread: 2^32 threads
    (1, 33, 16, 4, 1 << 27),    # single elements: 17 chunks, two threads each
    (0, 128, 64, 64, 1 << 23)])
def test_rotated_tokens(dtype, d, pairs, heads, tokens):
    lib = N.lib()
    rows, few = _heads(heads, d), _heads(heads, d)
    rot = N.Rotation(256, pairs, 256, False, False, 1.0, False)
    for batches, t in ((1, tokens), (2, tokens // 2)):
        assert lib.ojx_rotary(ctypes.byref(rows), None, batches, t, d, dtype, ctypes.byref(rot), 0, 1,
                              None) == -1
        assert lib.ojx_rotary(ctypes.byref(few), ctypes.byref(rows), batches, t, d, dtype, ctypes.byref(rot),
                              0, 1, None) == -1
    assert lib.ojx_kv8_rotate_append(P, P, P, 4, heads, 16, d, P, heads * d, d, P, heads * d, d, dtype, P,
                                     tokens, ctypes.byref(rows), ctypes.byref(rot), None) == -1
