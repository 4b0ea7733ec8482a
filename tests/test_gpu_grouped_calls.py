"""The expert products and the adapter projection in the settings that a program calls them in."""

import pytest

from gpu_util import as_np
from test_gpu_grouped import assert_close, make, offsets_of

pytestmark = pytest.mark.gpu


def test_training_through_an_autograd_function(pkg, orc, dev):
    """Leaves that require a gradient are refused, and an autograd function of the three products
    gives their gradients."""
    import torch
    counts, N, K = [50, 0, 33, 9], 96, 72
    x, w, dy = make(dev, counts, N, K, "float32", seed=21)
    off, hoff = offsets_of(counts, dev)
    x.requires_grad_(True), w.requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        pkg.grouped_matmul(x, w, off)

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w)
            return pkg.grouped_matmul(x, w, off)

        @staticmethod
        def backward(ctx, dy):
            x, w = ctx.saved_tensors
            dy = dy.contiguous()
            return pkg.grouped_matmul_grad_input(dy, w, off), \
                pkg.grouped_matmul_grad_weight(x, dy, off)

    dx, dw = torch.autograd.grad(Product.apply(x, w), (x, w), dy)
    hx, hw, hdy = as_np(x), as_np(w), as_np(dy)
    assert_close(dx, *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, "float32")
    assert_close(dw, *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(counts), "float32")
