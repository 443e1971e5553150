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
