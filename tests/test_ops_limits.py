"""Sizes at which the operators' index arithmetic would leave 32 bits: refused, or answered, without a device."""
import ctypes

import pytest

import hoard_amd as H

A = 0x10000  # an address that is aligned and never read: every call here returns before a launch


@pytest.mark.parametrize("call,args", [("gather", 4), ("combine", 5), ("combine_grad", 6)])
@pytest.mark.parametrize("n", [2**30 + 1, 2**31 - 7, 2**31 - 1])
def test_rows_of_too_many_columns(hlib, call, args, n):
    rc = getattr(hlib, "hoard_sort_" + call)(H.TYPE_BF16, 1, 1, n, *([A] * args), None)
    assert rc == H.ERR_INVALID and f"n {n}" in hlib.hoard_last_error().decode()
    assert getattr(hlib, "hoard_sort_" + call)(H.TYPE_BF16, 0, 1, 2**30, *([None] * args), None) == H.OK


@pytest.mark.parametrize("rows", [2**31 - 1, 2**31 - 1024, 2**31 - 256, 2**30 + 1])
@pytest.mark.parametrize("n", [1, 64, 1500, 16384])
def test_norm_workspace_of_many_rows(hlib, rows, n):
    a, need = H.NormArgs(H.TYPE_F16, H.TYPE_F16, H.GATE_NONE, 0, rows, n, 1e-6, 1.0, 0.0), ctypes.c_size_t()
    assert hlib.hoard_norm_workspace(ctypes.byref(a), ctypes.byref(need)) == H.OK
    assert 12 * n * 128 <= need.value <= 12 * n * 1024
    # short of that, the call is refused rather than launched
    a.r_out, a.w_pre, a.stats = A, A, A
    g = H.NormGrads(None, A, A, None, None, None, A)
    assert hlib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(g), A, need.value - 1, None) == H.ERR_INVALID


@pytest.mark.parametrize("n_mat", [2**30 + 1, 2**31 - 1])
def test_too_many_matrices(hlib, n_mat):
    w = ctypes.byref(H.Q4Matrix(A, A, None, 1, 32, 32, n_mat, H.TYPE_F16))
    assert hlib.hoard_q4_matmul_sorted(w, None, H.TYPE_BF16, 1, A, A, A, None) == H.ERR_UNSUPPORTED
    assert hlib.hoard_q4_matmul_ids(w, None, H.TYPE_BF16, 1, A, 1, A, A, None) == H.ERR_UNSUPPORTED
    assert f"n_mat {n_mat}" in hlib.hoard_last_error().decode()
