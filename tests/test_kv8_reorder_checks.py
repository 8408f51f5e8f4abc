"""What reordered requests and copied blocks refuse at the C ABI, before anything is launched; the
rule's own small cases."""

import ctypes

import reorder_plain as R
from ojasx_amd import _native as N


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = N.lib()
    P = ctypes.c_void_p(256)  # never read: every call is refused or has nothing to do
    good = [P, 3, P, 2, P, 4, 4, P, 5, P, 16, 9, P, P, P, P, P, P, None, 0, None]
    for i, value, code in ((1, -1, -1), (3, -1, -1), (5, 3, -1), (6, -1, -1), (8, -1, -1), (10, 24, -2),
                           (11, -1, -1), (11, 1 << 31, -1), (1, 1 << 31, -1), (0, None, -1),
                           (2, None, -1), (4, None, -1), (7, None, -1), (9, None, -1), (12, None, -1),
                           (13, None, -1), (14, None, -1), (15, None, -1), (16, None, -1),
                           (17, None, -1), (18, ctypes.c_void_p(8), -2), (19, 8, -1)):
        a = list(good)
        a[i] = value
        assert lib.ojx_kv8_reorder(*a) == code, (i, value)
    n = ctypes.c_size_t(7)
    size = lib.ojx_kv8_reorder_workspace_bytes
    assert size(2, 3, 4, 16, 9, ctypes.byref(n)) == 0 and n.value == 0
    assert size(4000, 4000, 400, 16, 10 ** 6, ctypes.byref(n)) == 0 and n.value > 4 * 4000 + 10 ** 6 // 4
    assert size(2, 3, 4, 17, 9, ctypes.byref(n)) == -2 and size(2, 3, 4, 16, 9, None) == -1
    big = list(good)
    big[3], big[1], big[5], big[6] = 4000, 4000, 400, 400   # needs a workspace
    assert lib.ojx_kv8_reorder(*big) == -1

    caches = (N.KV8Storage * 2)((256, 256, 256), (256, 256, 256))
    good = [caches, 2, 4, 2, 16, 80, P, P, 3, None]
    for i, value, code in ((0, None, -1), (1, -1, -1), (2, -1, -1), (3, 0, -1), (4, 20, -2), (5, 300, -2),
                           (6, None, -1), (7, None, -1), (8, -1, -1)):
        a = list(good)
        a[i] = value
        assert lib.ojx_kv8_copy_blocks(*a) == code, (i, value)
    bad = (N.KV8Storage * 2)((256, 256, 256), (256, 8, 256))
    assert lib.ojx_kv8_copy_blocks(bad, *good[1:]) == -2
    for i in (1, 2, 8):
        a = list(good)
        a[i] = 0
        assert lib.ojx_kv8_copy_blocks(*a) == 0


def test_the_rule():
    # two beams of row 0, none of row 1, which shared block 3
    out = R.reorder([0, 0], [20, 18], [[3, 4], [3, 5]], [9, 8], 2, 16, 10)
    assert out == ([[3, 4], [3, 5]], [20, 20], [9, 8] + [-1] * 8, 2, [-1, 4], [-1, 5])
    # all done
    out = R.reorder([-1, -1], [20, 18], [[3, 4], [3, 5]], [9, 8], 2, 16, 10)
    assert out[2] == [9, 8, 3, 4, 5] + [-1] * 5 and out[3] == 5 and out[1] == [0, 0]
