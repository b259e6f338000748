"""Argument checks of the operators with types and large class counts, without a GPU: the C entry
points refuse on the host, the wrappers refuse CPU tensors."""
import ctypes
import os

import pytest
import torch

BAD = ctypes.c_void_p(256)          # never dereferenced: every call below fails validation first
ODD = ctypes.c_void_p(257)


@pytest.fixture(scope="module")
def lib():
    from jittorgeometric_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from jittorgeometric_amd import build
        build.build()
    return _lib.load()


def test_grouped_rows_arguments(lib):
    n = ctypes.c_size_t(0)
    rows = lib.jgamd_grouped_rows
    for M, K, N, G in ((-1, 4, 4, 2), (5, 0, 4, 2), (5, 4, 0, 2), (5, 4, 4, 0), (5, (1 << 20) + 1, 4, 2), (5, 4, 4, 65536)):
        assert rows(BAD, BAD, BAD, BAD, BAD, M, K, N, G, 0, 0, None) == -2
        assert lib.jgamd_grouped_rows_weight_grad_workspace(M, K, N, G, ctypes.byref(n)) == -2
        assert lib.jgamd_grouped_rows_weight_grad(BAD, BAD, BAD, BAD, BAD, M, K, N, G, 0, BAD, 1 << 40, None) == -2
    assert rows(BAD, BAD, BAD, BAD, BAD, 5, 4, 4, 2, 7, 0, None) == -4
    assert rows(BAD, BAD, BAD, BAD, BAD, 5, 4, 4, 2, 0, 2, None) == -2
    assert rows(None, None, None, None, None, 0, 4, 4, 2, 0, 0, None) == 0
    for i in (0, 1, 3, 4):
        args = [BAD] * 5
        args[i] = None
        assert rows(*args, 5, 4, 4, 2, 0, 0, None) == -1
    for i in range(5):
        args = [BAD] * 5
        args[i] = ODD
        assert rows(*args, 5, 4, 4, 2, 1, 0, None) == -5
    assert rows(BAD, BAD, None, BAD, BAD, 2**31 - 1, 4, 1 << 20, 65535, 0, 0, None) == -2
    grad = lib.jgamd_grouped_rows_weight_grad
    assert lib.jgamd_grouped_rows_weight_grad_workspace(5, 4, 4, 2, None) == -1
    assert lib.jgamd_grouped_rows_weight_grad_workspace(100, 4, 4, 2, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.jgamd_grouped_rows_weight_grad_workspace(100_000, 64, 64, 9, ctypes.byref(n)) == 0 and 0 < n.value < 1 << 28
    assert lib.jgamd_grouped_rows_weight_grad_workspace(2**31 - 1, 1 << 10, 1 << 10, 65535, ctypes.byref(n)) == 0
    for i in range(4):
        args = [BAD] * 4
        args[i] = None
        assert grad(*args, None, 5, 4, 4, 2, 0, None, 0, None) == -1
        args[i] = ODD
        assert grad(*args, None, 5, 4, 4, 2, 1, None, 0, None) == -5
    assert grad(BAD, BAD, BAD, BAD, BAD, 100_000, 64, 64, 9, 0, None, 0, None) == -3
    assert grad(BAD, BAD, BAD, BAD, BAD, 100_000, 64, 64, 9, 0, BAD, 16, None) == -3
    assert grad(BAD, BAD, BAD, BAD, BAD, 100_000, 64, 64, 9, 0, ctypes.c_void_p(260), 1 << 40, None) == -5


def test_wrappers_refuse_cpu_tensors():
    from jittorgeometric_amd import JgamdError
    from jittorgeometric_amd.ops import grouped_rows
    with pytest.raises(JgamdError):
        grouped_rows(torch.zeros(4, 3), torch.zeros(2, 3, 5), torch.zeros(3, dtype=torch.int32))


def test_residual_norm_arguments(lib):
    n = ctypes.c_size_t(0)
    fwd, bwd = lib.jgamd_residual_norm_fwd, lib.jgamd_residual_norm_bwd
    for R, F in ((-1, 8), (5, 0), (5, 8193), (1 << 31, 8)):
        assert fwd(*[BAD] * 10, R, F, 1e-6, 0, None) == -2
        assert bwd(*[BAD] * 16, R, F, 0, BAD, 1 << 40, None) == -2
        assert lib.jgamd_residual_norm_bwd_workspace(R, F, ctypes.byref(n)) == -2
    assert lib.jgamd_residual_norm_bwd_workspace(5, 8, None) == -1
    assert fwd(*[BAD] * 10, 5, 8, 1e-6, 3, None) == -4
    assert bwd(*[BAD] * 16, 5, 8, 3, BAD, 1 << 40, None) == -4
    for i in (0, 5, 7):                                        # x, w, h
        args = [BAD] * 10
        args[i] = None
        assert fwd(*args, 5, 8, 1e-6, 0, None) == -1
    assert fwd(BAD, None, BAD, None, None, BAD, None, BAD, None, None, 5, 8, 1e-6, 0, None) == -1      # gate without y
    for i in range(10):
        args = [BAD] * 10
        args[i] = ODD
        assert fwd(*args, 5, 8, 1e-6, 1, None) == -5
    assert fwd(*[None] * 10, 0, 8, 1e-6, 0, None) == 0
    assert lib.jgamd_residual_norm_bwd_workspace(100_000, 256, ctypes.byref(n)) == 0 and 0 < n.value < 1 << 24
    for i in (0, 1, 2, 3, 4, 5, 6, 7):                         # an input that a gradient needs
        args = [BAD] * 16
        args[i] = None
        assert bwd(*args, 5, 8, 0, BAD, 1 << 40, None) == -1
    for i in range(16):
        args = [BAD] * 16
        args[i] = ODD
        assert bwd(*args, 5, 8, 1, BAD, 1 << 40, None) == -5
    assert bwd(*[BAD] * 16, 5, 8, 0, None, 0, None) == -3
    assert bwd(*[BAD] * 16, 5, 8, 0, BAD, 16, None) == -3
    assert bwd(*[BAD] * 16, 5, 8, 0, ctypes.c_void_p(260), 1 << 40, None) == -5


def test_norm_wrappers_refuse_cpu_tensors():
    from jittorgeometric_amd import JgamdError
    from jittorgeometric_amd.nn import residual_norm, rms_norm
    with pytest.raises(JgamdError):
        rms_norm(torch.zeros(4, 3), torch.ones(3))
    with pytest.raises(JgamdError):
        residual_norm(torch.zeros(4, 3), torch.zeros(4, 3), torch.ones(3))


def test_linear_cross_entropy_arguments(lib):
    n = ctypes.c_size_t(0)
    fwd, bwd, size = (lib.jgamd_linear_cross_entropy_fwd, lib.jgamd_linear_cross_entropy_bwd,
                      lib.jgamd_linear_cross_entropy_workspace)
    for V, F, C in ((-1, 8, 9), (5, 0, 9), (5, 8, 0), (1 << 31, 8, 9), (5, (1 << 20) + 1, 9), (5, 8, 2**31 - 1)):
        assert size(V, F, C, 0, 0, ctypes.byref(n)) == -2
        assert fwd(*[BAD] * 4, 1, V, F, C, 0, 1, *[BAD] * 4, 1 << 40, None) == -2
        assert bwd(*[BAD] * 4, 1, *[BAD] * 3, V, F, C, 0, 1, *[BAD] * 4, 1 << 40, None) == -2
    assert size(5, 8, 9, 0, 0, None) == -1
    assert size(5, 8, 9, 2, 0, ctypes.byref(n)) == -4
    assert fwd(*[BAD] * 4, 1, 5, 8, 9, 0, 3, *[BAD] * 4, 1 << 40, None) == -2
    assert fwd(*[BAD] * 4, 1, 5, 8, 9, 2, 1, *[BAD] * 4, 1 << 40, None) == -4
    for i in (0, 1, 3, 9, 10, 11):                      # x, w, labels; loss, count, lse
        a = [BAD] * 4 + [1, 5, 8, 9, 0] + [BAD] * 3
        a[i] = None
        assert fwd(*a[:9], 1, *a[9:], BAD, 1 << 40, None) == -1
        if i < 4:
            assert bwd(*a[:4], 1, *[BAD] * 3, 5, 8, 9, 0, 1, *[BAD] * 4, 1 << 40, None) == -1
    for i in range(4):
        a = [BAD] * 4
        a[i] = ODD
        assert fwd(*a, 1, 5, 8, 9, 1, 1, *[BAD] * 4, 1 << 40, None) == -5
        assert bwd(*a, 1, *[BAD] * 3, 5, 8, 9, 1, 1, *[BAD] * 4, 1 << 40, None) == -5
    assert fwd(*[BAD] * 4, 1, 5, 8, 9, 0, 1, *[BAD] * 3, None, 0, None) == -3
    assert fwd(*[BAD] * 4, 1, 5, 8, 9, 0, 1, *[BAD] * 4, 16, None) == -3
    assert fwd(*[BAD] * 4, 1, 5, 8, 9, 0, 1, *[BAD] * 3, ctypes.c_void_p(260), 1 << 40, None) == -5
    assert bwd(*[BAD] * 4, 1, *[BAD] * 3, 5, 8, 9, 0, 1, BAD, None, BAD, BAD, 1 << 40, None) == -1      # db without dw
    assert bwd(*[BAD] * 4, 1, *[BAD] * 3, 5, 8, 9, 0, 1, *[BAD] * 3, None, 0, None) == -3
    assert bwd(*[BAD] * 4, 1, *[BAD] * 3, 5, 8, 9, 0, 1, *[BAD] * 4, 16, None) == -3
    assert bwd(*[BAD] * 4, 1, *[BAD] * 3, 5, 8, 9, 0, 1, None, None, None, None, 0, None) == 0
    for back in (0, 1):
        assert size(0, 8, 9, 0, back, ctypes.byref(n)) == 0
    # the scratch does not grow with rows * classes
    assert size(1 << 20, 256, 1 << 20, 1, 1, ctypes.byref(n)) == 0 and n.value < 3 << 30
    assert size(1 << 20, 256, 1 << 20, 1, 0, ctypes.byref(n)) == 0 and n.value < 1 << 30


def test_sizes_past_32_bits_are_refused():
    from jittorgeometric_amd import JgamdError, _lib
    _lib.check_int32("f", torch.empty(2**31 - 1, 0), torch.empty(()))
    with pytest.raises(JgamdError):
        _lib.check_int32("f", torch.empty(3), torch.empty(0, 2**31))
