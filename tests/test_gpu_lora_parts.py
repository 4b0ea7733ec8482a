"""What the adapter projection's intermediate s_a A_a x carries on the tensor cores, where it is
the sum of two 16-bit parts above eight rows: overflow, infinities and precision.

An entry v = hi + lo + e: lo is at most half a step of hi, 2^-8 |v| in bfloat16 and 2^-11 |v| in
float16, and rounded to half a step of its own, so |e| <= 2^-16 |v| and 2^-22 |v|, in float16 not
below half its smallest step, 2^-25."""

import numpy as np
import pytest

from gpu_util import as_np, torch_dtype
from test_gpu_grouped import HALF_STEP

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


PART = {"float16": 2.0 ** -22, "bfloat16": 2.0 ** -16}
SMALLEST = {"float16": 2.0 ** -25, "bfloat16": 0.0}


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("r", [8, 40])
@pytest.mark.parametrize("T,N,kind", FORMS)
def test_what_the_second_part_holds(pkg, dev, dtype_name, T, N, kind, r):
    """Pairs of entries that are equal but for bits below the first part, with B = 1 and -1: y is
    what the second parts hold, and the first cancel.  (x[t] = (1, s), A = (a, b): t = a + s b,
    exact in float32.)"""
    import torch
    step = 2.0 ** -11 if dtype_name == "float16" else 2.0 ** -8
    d = call(dev, dtype_name, T, N, kind, r=r)
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: (torch.rand(*s, device=dev, generator=g) + 1).to(d["x"].dtype)
    d["x"][:, 0], d["x"][:, 1] = 1.0, step
    a = rnd(3, r // 2)
    d["lora_a"][:, 0::2, 0], d["lora_a"][:, 1::2, 0] = a, a
    # Below half a step of a, and further below for the odd entries.
    d["lora_a"][:, 0::2, 1], d["lora_a"][:, 1::2, 1] = rnd(3, r // 2) / 8 + 0.6, rnd(3, r // 2) / 8 + 0.4
    sign = torch.where(torch.arange(N, device=dev) % 3 == 0, -1.0, 1.0)[None, :, None]
    d["lora_b"][:, :, 0::2], d["lora_b"][:, :, 1::2] = sign, -sign
    y = as_np(pkg.lora_matmul(**d))
    ids, A, B = d["adapter_ids"].cpu().numpy(), as_np(d["lora_a"]), as_np(d["lora_b"])
    t = A[:, :, 0] + step * A[:, :, 1]
    exact = np.einsum("lnr,lr->ln", B, t)
    mag = np.abs(t).sum(1)[:, None]
    acc = np.maximum(PART[dtype_name] * np.abs(t), SMALLEST[dtype_name]).sum(1)[:, None]
    acc = acc + (2 * r + 4) * 2.0 ** -23 * mag
    tol = acc + HALF_STEP[dtype_name] * (np.abs(exact) + acc)
    rows = ids >= 0
    assert (np.abs(y[rows] - exact[ids[rows]]) <= tol[ids[rows]]).all()
    assert not y[~rows].any()
    # The test can tell: without the second parts y would be 0, outside the tolerance everywhere.
    assert bool((np.abs(exact) > tol).all())


@pytest.mark.parametrize("T,N,kind", FORMS[1:])
@pytest.mark.parametrize("top", [2.0 ** -8, 1.0, 2.0 ** 14])
def test_small_entries_beside_a_large_one(pkg, dev, T, N, kind, top):
    """float16: an entry far below its row's largest keeps 2^-25, whatever its own size."""
    d = call(dev, "float16", T, N, kind)
    small = 2.0 ** -20 * (1 + 2.0 ** -8)
    d["x"][:, 0], d["x"][:, 1] = 1.0, 2.0 ** -10
    d["lora_a"][:, 0, 0] = top
    d["lora_a"][:, 1, 1] = small * 2.0 ** 10
    d["lora_b"][:, :, 1] = 2.0 ** 12
    y = as_np(pkg.lora_matmul(**d))
    rows = has_adapter(d).cpu().numpy()
    exact, tol = small * 2.0 ** 12, 2.0 ** -25 * 2.0 ** 12
    assert (np.abs(y[rows] - exact) <= tol + HALF_STEP["float16"] * (exact + tol)).all()
    assert not y[~rows].any()
