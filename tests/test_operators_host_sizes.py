"""Sizes that the class head refuses on the host, without a GPU."""
import ctypes
import os

BAD = ctypes.c_void_p(256)          # never dereferenced: every call below fails validation first


def test_rows_past_what_a_launch_counts():
    from jittorgeometric_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from jittorgeometric_amd import build
        build.build()
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    for V in (2**31 - 1, 2**31 - 255):
        assert lib.jgamd_linear_cross_entropy_workspace(V, 8, 9, 1, 0, ctypes.byref(n)) == -2
        assert lib.jgamd_linear_cross_entropy_fwd(*[BAD] * 4, 1, V, 8, 9, 1, 1, *[BAD] * 4, 1 << 62, None) == -2
        assert lib.jgamd_linear_cross_entropy_bwd(*[BAD] * 4, 1, *[BAD] * 3, V, 8, 9, 1, 1, *[BAD] * 4, 1 << 62, None) == -2
    assert lib.jgamd_linear_cross_entropy_workspace(2**31 - 256, 8, 9, 1, 0, ctypes.byref(n)) == 0
