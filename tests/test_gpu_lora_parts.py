"""What the adapter projection's intermediate s_a A_a x carries on the tensor cores, where it is
the sum of two 16-bit parts above eight rows: overflow and infinities."""

import numpy as np
import pytest

from gpu_util import torch_dtype

pytestmark = pytest.mark.gpu

# Rows and features that reach every kernel: one launch, the streaming kernel, pairs of tiles with
# sixteen rows of one adapter together ("runs") and apart.
FORMS = [(3, 64, "one"), (9, 64, "one"), (100, 136, "mixed"), (2048, 2048, "runs"),
         (2048, 2048, "mixed")]


def call(dev, dtype_name, T, N, kind, K=64, r=8, L=3, scale=1.0):
    """All zeros; every second adapter-less row only in mixed batches."""
    import torch
    dt = torch_dtype(dtype_name)
    z = lambda *s: torch.zeros(*s, device=dev, dtype=dt)
    ids = {"one": np.zeros(T), "runs": np.arange(T) * L // T, "mixed": np.arange(T) % (L + 1) - 1}
    return dict(x=z(T, K), weight=z(N, K), lora_a=z(L, r, K), lora_b=z(L, N, r),
                adapter_ids=torch.as_tensor(ids[kind], dtype=torch.int32).to(dev),
                scales=torch.full((L,), scale, device=dev))


def has_adapter(d):
    return d["adapter_ids"] >= 0


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("T,N,kind", FORMS)
def test_infinite_intermediate(pkg, dev, dtype_name, T, N, kind):
    """scale * (A x) past float32: infinite, with the sign of B; beside finite entries of the other
    sign, past the 16-bit types' range as well, it stays that infinity."""
    inf = float("inf")
    d = call(dev, dtype_name, T, N, kind, scale=3e38)
    d["x"][:, 0], d["x"][:, 1] = 64.0, 2.0 ** -24
    d["lora_a"][:, 2, 0] = 1.0             # 64 * 3e38
    d["lora_b"][:, ::2, 2], d["lora_b"][:, 1::2, 2] = 1.0, -0.5
    y = pkg.lora_matmul(**d)
    rows = has_adapter(d)
    assert (y[rows][:, ::2] == inf).all() and (y[rows][:, 1::2] == -inf).all()
    assert (y[~rows] == 0).all()
    d["lora_a"][:, 5, 1] = 2.0 ** -14      # 2^-38 * 3e38, about 2^90
    d["lora_b"][:, ::2, 5], d["lora_b"][:, 1::2, 5] = -1.0, 1.0
    y = pkg.lora_matmul(**d)
    assert (y[rows][:, ::2] == inf).all() and (y[rows][:, 1::2] == -inf).all()
    assert (y[~rows] == 0).all()


@pytest.mark.parametrize("T,N,kind", FORMS)
def test_intermediate_between_the_largest_bfloat16_and_float32(pkg, dev, T, N, kind):
    """1.5 * 2^119 above the largest bfloat16, which would round to infinity as one part."""
    d = call(dev, "bfloat16", T, N, kind)
    top = (2 - 2.0 ** -7) * 2.0 ** 127
    d["x"][:, :2] = 1.0
    d["lora_a"][:, 0, 0], d["lora_a"][:, 0, 1] = top, 1.5 * 2.0 ** 119
    d["lora_b"][:, :, 0] = 2.0 ** -100
    y = pkg.lora_matmul(**d)
    rows = has_adapter(d)
    exact = (top + 1.5 * 2.0 ** 119) * 2.0 ** -100
    assert ((y[rows].double() - exact).abs() <= exact * 2.0 ** -8).all() and (y[~rows] == 0).all()
