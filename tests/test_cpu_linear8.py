"""Refusals of the 8-bit products of tokens that need no GPU."""
import ctypes

import pytest

import nhip

P = ctypes.c_void_p
ONE = 4096  # stands for a device pointer: none of these calls gets as far as using it


def create(experts=1, n=8, k=16, weight=ONE, is_i8=1, scale=ONE, bias=None, act=0):
    h = P()
    st = nhip.load().nhip_linear8_create(experts, n, k, weight, is_i8, scale, bias, act, None, ctypes.byref(h))
    assert not h.value and nhip.load().nhip_last_error()
    return st


@pytest.mark.parametrize("change,status", [
    (dict(experts=0), 2), (dict(n=0), 2), (dict(k=-1), 2), (dict(k=131073), 2), (dict(act=nhip.ACT_SIGMOID), 7),
    (dict(experts=2 ** 20, n=2 ** 20), 4), (dict(weight=None), 1), (dict(scale=None), 1), (dict(is_i8=0), 3),
    (dict(is_i8=0, scale=None, weight=ONE + 2), 3), (dict(scale=ONE + 2), 3), (dict(bias=ONE + 1), 3)])
def test_create(change, status):
    assert create(**change) == status


def test_calls_without_a_plan():
    lib, n = nhip.load(), ctypes.c_uint64()
    assert lib.nhip_linear8_create(1, 8, 16, ONE, 1, ONE, None, 0, None, None) == 1
    assert lib.nhip_linear8_workspace_size(None, 0, 1, ctypes.byref(n)) == 1
    assert lib.nhip_linear8_forward(None, ONE, 0, 1, 16, None, ONE, ONE, 1 << 20, None) == 1
    assert lib.nhip_linear8_destroy(None) == 0
