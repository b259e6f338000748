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
