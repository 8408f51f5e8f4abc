"""What the rotated append refuses at the C ABI, before anything is launched."""

import ctypes
import math

from ojasx_amd import _native as N


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = N.lib()
    P = ctypes.c_void_p(256)  # never read: every call is refused or has nothing to do

    def call(i=None, value=None, rows=None, rot=None):
        q = N.RotaryRows(**{**dict(x=256, y=256, x_batch=0, x_token=480, x_head=80, y_batch=0,
                                   y_token=480, y_head=80, heads=6), **(rows or {})})
        r = N.Rotation(**{**dict(rates=256, pairs=40, positions=256, positions64=0, interleaved=0,
                                 gain=1.0, inverse=0), **(rot or {})})
        a = [P, P, P, 4, 2, 16, 80, P, 160, 80, P, 160, 80, 2, P, 3, ctypes.byref(q), ctypes.byref(r),
             None]
        if i is not None:
            a[i] = value
        return lib.ojx_kv8_rotate_append(*a)

    for i, value, code in ((3, -1, -1), (4, 0, -1), (5, 20, -2), (6, 0, -2), (6, 257, -2), (6, 79, -2),
                           (13, 3, -3), (15, -1, -1), (7, None, -1), (8, -1, -1), (14, None, -1),
                           (0, None, -1), (0, ctypes.c_void_p(8), -2), (17, None, -1)):
        assert call(i, value) == code, (i, value)
    for rows, code in ((dict(heads=-1), -1), (dict(x=0), -1), (dict(y=0), -1), (dict(x_token=-1), -1),
                       (dict(x=257), -2)):
        assert call(rows=rows) == code, rows
    for rot, code in ((dict(pairs=0), -2), (dict(pairs=41), -2), (dict(inverse=1), -1),
                      (dict(gain=math.inf), -1), (dict(positions=0), -1), (dict(rates=0), -1)):
        assert call(rot=rot) == code, rot
    assert call(15, 0) == 0
