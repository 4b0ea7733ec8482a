"""CPU tests of the error query of the expert products and the adapter projection."""

import ctypes


def test_no_error_before_any_call(pkg):
    assert pkg.take_device_error() == 0
    code = ctypes.c_int32(7)
    assert pkg.lib().moe_b200_take_device_error(ctypes.byref(code)) == pkg.OK and code.value == 0


def test_query_needs_somewhere_to_write(pkg):
    assert pkg.lib().moe_b200_take_device_error(None) == pkg.INVALID_ARGUMENT
    assert b"take_device_error" in pkg.lib().moe_b200_last_error()
