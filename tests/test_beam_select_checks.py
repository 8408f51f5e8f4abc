"""What the selection of beams refuses at the C ABI, before anything is launched."""

import ctypes

from ojasx_amd import _native as N


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = N.lib()
    P = ctypes.c_void_p(256)  # never read: every call is refused or has nothing to do
    n = ctypes.c_size_t(7)
    size = 2 * 4 * (16 + 8 * 8)
    good = [P, 100, 2, 4, 100, 2, P, P, 0, 8, P, P, P, P, size, None]

    def call(**change):
        a = list(good)
        for i, v in change.items():
            a[int(i[1:])] = v
        return lib.ojx_beam_select(*a)

    for i, value, code in ((1, 99, -1), (2, -1, -1), (2, 1 << 30, -1), (3, 0, -1), (3, 65, -1),
                           (4, 0, -1), (5, 3, -3), (8, -1, -1), (8, 100, -1), (9, 0, -1), (9, 65, -1),
                           (0, None, -1), (6, None, -1), (10, None, -1), (11, None, -1), (12, None, -1),
                           (13, None, -1), (13, ctypes.c_void_p(8), -2), (14, size - 1, -1),
                           (0, ctypes.c_void_p(257), -2), (6, ctypes.c_void_p(258), -2)):
        assert call(**{f"_{i}": value}) == code, (i, value)
    assert call(_13=None, _14=0) == -1
    assert call(_3=1, _4=5, _1=5, _9=6) == -1        # more than there are
    assert call(_2=0, _13=None, _14=0) == 0
    bad = lib.ojx_beam_select_workspace_bytes
    assert bad(2, 4, 100, 8, 2, None) == -1 and bad(2, 4, 100, 8, 7, ctypes.byref(n)) == -3
    assert bad(2, 4, 100, 8, 2, ctypes.byref(n)) == 0 and n.value == size
    assert bad(0, 4, 100, 8, 2, ctypes.byref(n)) == 0 and n.value == 0
