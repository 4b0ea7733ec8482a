"""CPU tests of the expert products and the adapter projection: argument checks of the C
entries and of their Python wrappers, and the float64 oracle's known answers.  A refused call
returns before any CUDA call, so these need no GPU."""

import ctypes

import numpy as np
import pytest

BUF = 1 << 20      # a non-NULL, well aligned address; refused calls never read it
SZ = ctypes.c_size_t


def _fwd(pkg, dtype=None, rows=4, n=16, k=16, E=2, x=BUF, w=BUF, off=BUF, y=BUF):
    return pkg.lib().moe_b200_grouped_matmul(pkg.FLOAT16 if dtype is None else dtype, rows, n, k,
                                             E, x, w, off, y, None)


def _gin(pkg, dtype=None, rows=4, n=16, k=16, E=2, x=BUF, w=BUF, off=BUF, y=BUF):
    return pkg.lib().moe_b200_grouped_matmul_grad_input(
        pkg.FLOAT16 if dtype is None else dtype, rows, n, k, E, x, w, off, y, None)


def _gw(pkg, dtype=None, rows=4, n=16, k=16, E=2, x=BUF, w=BUF, off=BUF, y=BUF, ws=BUF,
        nbytes=1 << 30):
    return pkg.lib().moe_b200_grouped_matmul_grad_weight(
        pkg.FLOAT16 if dtype is None else dtype, rows, n, k, E, x, w, off, y, ws, nbytes, None)


def _lora(pkg, dtype=None, rows=4, n=16, k=16, L=2, r=8, ptrs=(BUF,) * 7, ws=BUF,
          nbytes=1 << 30):
    return pkg.lib().moe_b200_lora_matmul(pkg.FLOAT16 if dtype is None else dtype, rows, n, k, L,
                                          r, *ptrs, ws, nbytes, None)


@pytest.mark.parametrize("call", [_fwd, _gin, _gw])
@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(n=0), dict(k=0), dict(n=(1 << 20) + 1),
    dict(k=(1 << 20) + 1), dict(E=0), dict(E=257), dict(x=None), dict(w=None), dict(off=None),
    dict(y=None), dict(x=BUF + 1), dict(y=BUF + 1), dict(off=BUF + 2),
])
def test_grouped_refusals(pkg, call, kw):
    assert call(pkg, **kw) == pkg.INVALID_ARGUMENT
    assert b"grouped_matmul" in pkg.lib().moe_b200_last_error()


@pytest.mark.parametrize("call", [_fwd, _gin, _gw, _lora])
def test_unsupported_types(pkg, call):
    assert call(pkg, dtype=pkg.UINT8) == pkg.NOT_IMPLEMENTED
    assert call(pkg, dtype=99) == pkg.NOT_IMPLEMENTED


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(n=0), dict(k=0), dict(L=0), dict(r=0), dict(r=257),
    *[dict(ptrs=(BUF,) * i + (None,) + (BUF,) * (6 - i)) for i in range(7)],
    dict(ptrs=(BUF + 1,) + (BUF,) * 6), dict(ptrs=(BUF,) * 4 + (BUF + 2,) + (BUF,) * 2),
    dict(ws=None), dict(ws=BUF + 16), dict(nbytes=0),
])
def test_lora_refusals(pkg, kw):
    assert _lora(pkg, **kw) == pkg.INVALID_ARGUMENT
    assert b"lora_matmul" in pkg.lib().moe_b200_last_error()


def test_no_rows_is_no_work(pkg):
    """Zero rows: nothing to do, and no buffer is needed."""
    assert _fwd(pkg, rows=0, x=None, y=None, off=None, w=None) == pkg.OK
    assert _gin(pkg, rows=0, x=None, y=None, off=None, w=None) == pkg.OK
    assert _lora(pkg, rows=0, ptrs=(None,) * 7, ws=None, nbytes=0) == pkg.OK
    assert _gw(pkg, rows=0, y=None) == pkg.INVALID_ARGUMENT  # zeros have to go somewhere


def test_workspace_sizes(pkg):
    n = SZ()
    L = pkg.lib()
    assert L.moe_b200_lora_matmul_workspace_size(pkg.BFLOAT16, 100, 16, ctypes.byref(n)) == pkg.OK
    assert n.value >= 100 * 16 * 4
    assert _lora(pkg, rows=100, r=16, nbytes=n.value - 1) == pkg.INVALID_ARGUMENT
    assert L.moe_b200_lora_matmul_workspace_size(pkg.BFLOAT16, 100, 0, ctypes.byref(n)) == \
        pkg.INVALID_ARGUMENT
    assert L.moe_b200_lora_matmul_workspace_size(pkg.BFLOAT16, 100, 16, None) == \
        pkg.INVALID_ARGUMENT
    f = L.moe_b200_grouped_matmul_grad_weight_workspace_size
    assert f(pkg.BFLOAT16, 64, 64, 8, ctypes.byref(n)) == pkg.OK
    if n.value:
        assert _gw(pkg, dtype=pkg.BFLOAT16, n=64, k=64, E=8, nbytes=n.value - 1) == \
            pkg.INVALID_ARGUMENT
        assert _gw(pkg, dtype=pkg.BFLOAT16, n=64, k=64, E=8, ws=None) == pkg.INVALID_ARGUMENT
        assert _gw(pkg, dtype=pkg.BFLOAT16, n=64, k=64, E=8, ws=BUF + 16) == pkg.INVALID_ARGUMENT
    assert f(pkg.BFLOAT16, 64, 64, 0, ctypes.byref(n)) == pkg.INVALID_ARGUMENT
    assert f(pkg.BFLOAT16, 64, 64, 8, None) == pkg.INVALID_ARGUMENT


def test_wrappers_refuse_host_tensors(pkg):
    import torch
    x, w = torch.zeros(4, 16), torch.zeros(2, 8, 16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.grouped_matmul(x, w, off)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.grouped_matmul_grad_input(torch.zeros(4, 8), w, off)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.grouped_matmul_grad_weight(x, torch.zeros(4, 8), off)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.lora_matmul(x, torch.zeros(8, 16), torch.zeros(1, 4, 16), torch.zeros(1, 8, 4),
                        torch.zeros(4, dtype=torch.int32), torch.ones(1))
    with pytest.raises(ValueError, match="dimensions"):
        pkg.grouped_matmul(torch.zeros(4), w, off)
    with pytest.raises(ValueError, match="dimensions"):
        pkg.lora_matmul(x, torch.zeros(8, 16), torch.zeros(4, 16), torch.zeros(1, 8, 4),
                        torch.zeros(4, dtype=torch.int32), torch.ones(1))


def test_oracle_known_answers(orc):
    x = np.array([[1., 2.], [3., 4.], [5., 6.]])
    w = np.array([[[1., 0.], [0., 1.], [1., 1.]], [[2., 0.], [0., 0.], [0., -1.]]])
    off = [0, 1, 2]  # the third row belongs to no expert
    y, mag = orc.grouped_matmul(x, w, off)
    np.testing.assert_array_equal(y[:2], [[1, 2, 3], [6, 0, -4]])
    assert np.isnan(y[2]).all()
    np.testing.assert_array_equal(mag[:2], [[1, 2, 3], [6, 0, 4]])
    dx, _ = orc.grouped_matmul_grad_input(y[:2], w, off)
    np.testing.assert_array_equal(dx, [[4, 5], [12, 4]])
    dw, _ = orc.grouped_matmul_grad_weight(x[:2], y[:2], off)
    np.testing.assert_array_equal(dw[0], [[1, 2], [2, 4], [3, 6]])
    np.testing.assert_array_equal(dw[1], [[18, 24], [0, 0], [-12, -16]])
    dw, _ = orc.grouped_matmul_grad_weight(x[:2], y[:2], [0, 2, 2])
    assert not dw[1].any()
    y, _, _ = orc.lora_matmul(x, np.eye(2), [[[1., 1.]]], [[[1.], [2.]]], [0, -1, 7], [0.5])
    np.testing.assert_array_equal(y, [[2.5, 5.0], [3, 4], [5, 6]])


# Buffers of 4 rows, 16 x 16 and two groups or adapters, far apart but for the pair under test.
FAR = [BUF + (i << 16) for i in range(8)]


def _moved(i, to):
    return [to if j == i else q for j, q in enumerate(FAR)]


@pytest.mark.parametrize("call", [_fwd, _gin])
@pytest.mark.parametrize("other,last", [("x", 4 * 16 * 2 - 16), ("w", 2 * 16 * 16 * 2 - 16),
                                        ("off", 8)])
def test_products_refuse_overlapping_output(pkg, call, other, last):
    at = dict(x=FAR[0], w=FAR[1], off=FAR[2])
    for y in (at[other], at[other] + last):
        assert call(pkg, y=y, **at) == pkg.INVALID_ARGUMENT
        assert b"overlap" in pkg.lib().moe_b200_last_error()


@pytest.mark.parametrize("other,last", [("x", 4 * 16 * 2 - 16), ("w", 4 * 16 * 2 - 16),
                                        ("off", 8)])
def test_grad_weight_refuses_overlapping_buffers(pkg, other, last):
    at = dict(x=FAR[0], w=FAR[1], off=FAR[2])  # (`w` is where this call takes dy)
    for y in (at[other], at[other] + last, FAR[4]):
        assert _gw(pkg, y=y, ws=FAR[4], **at) == pkg.INVALID_ARGUMENT
        assert b"overlap" in pkg.lib().moe_b200_last_error()
    assert _gw(pkg, y=FAR[3], ws=at[other], **at) == pkg.INVALID_ARGUMENT
    assert b"overlap" in pkg.lib().moe_b200_last_error()


@pytest.mark.parametrize("i", [0, 1, 2, 3, 4, 5, 7])
def test_lora_refuses_overlapping_buffers(pkg, i):
    # x, weight, lora_a, lora_b, adapter_ids, scales, y (6), workspace
    at = _moved(6, FAR[i])
    assert _lora(pkg, ptrs=tuple(at[:7]), ws=at[7]) == pkg.INVALID_ARGUMENT
    assert b"overlap" in pkg.lib().moe_b200_last_error()
    if i < 6:
        at = _moved(7, FAR[i])
        assert _lora(pkg, ptrs=tuple(at[:7]), ws=at[7]) == pkg.INVALID_ARGUMENT
        assert b"overlap" in pkg.lib().moe_b200_last_error()
