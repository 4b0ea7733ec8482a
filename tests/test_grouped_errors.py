"""CPU tests of the expert products and the adapter projection: the error query, and arguments
that require a gradient."""

import ctypes

import pytest


def test_no_error_before_any_call(pkg):
    assert pkg.take_device_error() == 0
    code = ctypes.c_int32(7)
    assert pkg.lib().moe_b200_take_device_error(ctypes.byref(code)) == pkg.OK and code.value == 0


def test_query_needs_somewhere_to_write(pkg):
    assert pkg.lib().moe_b200_take_device_error(None) == pkg.INVALID_ARGUMENT
    assert b"take_device_error" in pkg.lib().moe_b200_last_error()


def _calls(pkg, torch):
    """Every call on host tensors, which it refuses behind the check of gradients."""
    t = lambda *s: torch.zeros(*s)
    off, ids = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    return {
        "grouped_matmul": (pkg.grouped_matmul, [t(4, 16), t(2, 8, 16), off, t(4, 8)], (0, 1, 3)),
        "grouped_matmul_grad_input": (pkg.grouped_matmul_grad_input,
                                      [t(4, 8), t(2, 8, 16), off, t(4, 16)], (0, 1, 3)),
        "grouped_matmul_grad_weight": (pkg.grouped_matmul_grad_weight,
                                       [t(4, 16), t(4, 8), off, t(2, 8, 16)], (0, 1, 3)),
        "lora_matmul": (pkg.lora_matmul, [t(4, 16), t(8, 16), t(2, 4, 16), t(2, 8, 4), ids, t(2),
                                          t(4, 8)], (0, 1, 2, 3, 5, 6)),
    }


@pytest.mark.parametrize("name", ["grouped_matmul", "grouped_matmul_grad_input",
                                  "grouped_matmul_grad_weight", "lora_matmul"])
def test_arguments_that_require_a_gradient(pkg, name):
    """Refused while gradients are recorded, and only then: a result without history would train
    wrongly and say nothing."""
    import torch
    call, args, floats = _calls(pkg, torch)[name]
    for i in floats:
        args[i].requires_grad_(True)
        with pytest.raises(ValueError, match=f"{name}: .* gradient"):
            call(*args)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call(*args)
        args[i].requires_grad_(False)
    with pytest.raises(ValueError, match="CUDA"):
        call(*args)
