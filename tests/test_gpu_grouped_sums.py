"""Long contractions of the expert products and the adapter projection.

Tensor cores (16-bit types).  Products of same-signed operands, so that nothing averages out.
One MMA step adds sixteen products to the running fp32 sum and loses at most two of its units
in the last place (the products are aligned to the sum and cut off), 2^-22 of it.  An accumulator
takes at most 16384 entries, 1024 steps, before it is added to a sum of its own: 2^-12 of the
magnitudes, whatever the length, and half a step of the output type.

FFMA kernels (float32).  512 products per running sum lose half a step each; the sums of those
sums lose at most 64 more on their way (2^20 entries over 32 lanes) or, in the tiles, carry their
rounding errors along; then up to five additions across lanes and four across a cluster.
"""

import numpy as np
import pytest

from gpu_util import torch_dtype
from test_gpu_grouped import FLOOR, HALF_STEP

pytestmark = pytest.mark.gpu

SEGMENT = 2.0 ** -12
FFMA = (512 + 64 + 5 + 4) * 2.0 ** -24


def positive(dev, shape, scale, dtype_name, seed):
    """Uniform in [1, 2) times a power of two."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.rand(shape, device=dev, generator=g) + 1).mul_(scale).to(torch_dtype(dtype_name))


def assert_sums(got, exact, dtype_name, acc=SEGMENT):
    """`exact`: float64, all positive, so it is also its own sum of magnitudes."""
    err = (got.double() - exact).abs()
    tol = exact * (acc + HALF_STEP[dtype_name] * (1 + acc)) + FLOOR[dtype_name]
    assert bool((err <= tol).all()), f"{float((err / exact).max())} of the value"


def offsets(dev, counts):
    import torch
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=dev)


# Rows, features: few rows in tiles of 16, 128 and 256 rows, then pairs of tiles for several
# rounds of the GPU.
@pytest.mark.parametrize("counts,feat,con", [
    ([3], 72, 524328), ([2, 0, 5], 136, 262152), ([100], 64, 524328), ([200], 64, 524328),
    ([4000], 1800, 131080)])
@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
def test_long_contractions(pkg, dev, dtype_name, counts, feat, con):
    rows, E = sum(counts), len(counts)
    scale = 2.0 ** -8
    off = offsets(dev, counts)
    a = positive(dev, (rows, con), scale, dtype_name, 1)
    w = positive(dev, (E, feat, con), 1.0, dtype_name, 2)
    y = pkg.grouped_matmul(a, w, off)
    at = np.cumsum([0] + counts)
    for e in range(E):
        s = slice(at[e], at[e + 1])
        assert_sums(y[s], a[s].double() @ w[e].double().t(), dtype_name)
    del w, y
    w = positive(dev, (E, con, feat), 1.0, dtype_name, 3)
    dx = pkg.grouped_matmul_grad_input(a, w, off)
    for e in range(E):
        s = slice(at[e], at[e + 1])
        assert_sums(dx[s], a[s].double() @ w[e].double(), dtype_name)


# Experts of several sums, of one, of a part of one and without rows follow each other, in
# several rounds of the GPU; then one tile with many.
@pytest.mark.parametrize("counts,N,K", [
    ([40000, 0, 3, 16385, 70001], 1032, 1544), ([524325], 64, 72), ([16384, 32768, 16400], 520, 264)])
@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
def test_long_grad_weight(pkg, dev, dtype_name, counts, N, K):
    rows = sum(counts)
    off = offsets(dev, counts)
    x = positive(dev, (rows, K), 2.0 ** -8, dtype_name, 4)
    dy = positive(dev, (rows, N), 1.0, dtype_name, 5)
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)
    at = np.cumsum([0] + counts)
    for e, c in enumerate(counts):
        s = slice(at[e], at[e + 1])
        if c == 0:
            assert not dw[e].any()
        else:
            assert_sums(dw[e], dy[s].double().t() @ x[s].double(), dtype_name)


def test_long_grad_weight_of_a_large_call(pkg, dev):
    """Two experts of half a million and sixty thousand rows whose products nearly cancel."""
    import torch
    counts, N, K = [500_000, 60_000, 13], 256, 64
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(sum(counts), K, device=dev, generator=g).bfloat16()
    dy = torch.randn(sum(counts), N, device=dev, generator=g).bfloat16()
    dw = pkg.grouped_matmul_grad_weight(x, dy, offsets(dev, counts))
    at = np.cumsum([0] + counts)
    for e in range(3):
        s = slice(at[e], at[e + 1])
        exact = dy[s].double().t() @ x[s].double()
        mag = dy[s].double().abs().t() @ x[s].double().abs()
        assert ((dw[e].double() - exact).abs() <= exact.abs() * 2.0 ** -8 + mag * SEGMENT).all()


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
def test_sums_that_overflow_stay_infinite(pkg, dev, dtype_name):
    """An infinity or NaN in an early part of a long sum is still there at its end."""
    import torch
    R, N, K = 70000, 64, 64
    x = positive(dev, (R, K), 2.0 ** -8, dtype_name, 6)
    dy = positive(dev, (R, N), 1.0, dtype_name, 7)
    off = offsets(dev, [R])
    clean = pkg.grouped_matmul_grad_weight(x, dy, off)
    dy[100, 3], dy[40000, 5], dy[17, 7] = float("inf"), float("-inf"), float("nan")
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)[0]
    assert (dw[3] == float("inf")).all() and (dw[5] == float("-inf")).all() and dw[7].isnan().all()
    keep = torch.ones(N, dtype=torch.bool, device=dev)
    keep[[3, 5, 7]] = False
    assert torch.equal(dw[keep], clean[0][keep])


# One launch, the streaming kernel (tiles of 64 and 256 rows), pairs of tiles with runs of rows
# and with rows that follow several adapters.
@pytest.mark.parametrize("T,N,K,r,kind", [
    (4, 136, 262208, 16, "mixed"), (40, 136, 262208, 16, "mixed"), (200, 72, 262208, 24, "mixed"),
    (4000, 1800, 65608, 16, "runs"), (2100, 2304, 65608, 8, "mixed")])
@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
def test_long_adapter_sums(pkg, dev, dtype_name, T, N, K, r, kind):
    import torch
    L = 3
    ids = np.arange(T) % (L + 1) - 1 if kind == "mixed" else np.arange(T) // (T // 3 + 1)
    d = dict(x=positive(dev, (T, K), 1.0, dtype_name, 8),
             weight=positive(dev, (N, K), 2.0 ** -13, dtype_name, 9),
             lora_a=positive(dev, (L, r, K), 2.0 ** -13, dtype_name, 10),
             lora_b=positive(dev, (L, N, r), 2.0 ** -5, dtype_name, 11),
             adapter_ids=torch.as_tensor(ids, dtype=torch.int32).to(dev),
             scales=torch.tensor([0.5, 1.0, 2.0], device=dev))
    y = pkg.lora_matmul(**d)
    exact = d["x"].double() @ d["weight"].double().t()
    for a in range(L):
        rows = torch.as_tensor(ids == a, device=dev)
        t = d["x"][rows].double() @ d["lora_a"][a].double().t()
        exact[rows] += float(d["scales"][a]) * (t @ d["lora_b"][a].double().t())
    # t's own sum, its two 16-bit parts (2^-15) and the sum over the rank.
    assert_sums(y, exact, dtype_name, SEGMENT + 2.0 ** -15 + (r + 6) * 2.0 ** -23)


# 8 x 256 slices of 64 and one more: one CTA of a cluster of eight has a second segment (of one slice);
# a pair's second segment has 8 entries; an expert of 16383 rows has 255 slices, a step and a tail.
@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("T", [4, 9, 40, 100, 200])
def test_segments_of_some_ctas(pkg, dev, dtype_name, T):
    import torch
    con = 8 * 16384 + 64
    off = offsets(dev, [T])
    a, w = positive(dev, (T, con), 2.0 ** -8, dtype_name, 1), positive(dev, (1, 72, con), 1.0, dtype_name, 2)
    assert_sums(pkg.grouped_matmul(a, w, off), a.double() @ w[0].double().t(), dtype_name)
    wt = w.transpose(1, 2).contiguous()
    assert_sums(pkg.grouped_matmul_grad_input(a, wt, off), a.double() @ w[0].double().t(), dtype_name)
    lora_a = positive(dev, (2, 16, con), 2.0 ** -6, dtype_name, 3)
    lora_b = positive(dev, (2, 72, 16), 2.0 ** -4, dtype_name, 4)
    ids = torch.arange(T, dtype=torch.int32, device=dev) % 2
    y = pkg.lora_matmul(a, w[0], lora_a, lora_b, ids, torch.ones(2, device=dev))
    exact = a.double() @ w[0].double().t()
    for i in range(2):
        exact[i::2] += a[i::2].double() @ lora_a[i].double().t() @ lora_b[i].double().t()
    assert_sums(y, exact, dtype_name, SEGMENT + 2.0 ** -15 + 22 * 2.0 ** -23)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("con", [16384, 16392])
def test_pairs_at_the_end_of_a_segment(pkg, dev, dtype_name, con):
    T, N = 2048, 1800
    off = offsets(dev, [T])
    a, w = positive(dev, (T, con), 2.0 ** -8, dtype_name, 1), positive(dev, (1, N, con), 1.0, dtype_name, 2)
    assert_sums(pkg.grouped_matmul(a, w, off), a.double() @ w[0].double().t(), dtype_name)
    counts = [16383, 1, 16384, 16385, 32769, 0, 16400]
    x = positive(dev, (sum(counts), 72), 2.0 ** -8, dtype_name, 3)
    dy = positive(dev, (sum(counts), 136), 1.0, dtype_name, 4)
    dw = pkg.grouped_matmul_grad_weight(x, dy, offsets(dev, counts))
    at = np.cumsum([0] + counts)
    for e in range(len(counts)):
        s = slice(at[e], at[e + 1])
        assert_sums(dw[e], dy[s].double().t() @ x[s].double(), dtype_name)


LONG = 1 << 20


@pytest.mark.parametrize("c", [1 + 2.0 ** -13 - 2.0 ** -16, np.float32(1.3)])
def test_fp32_lanes(pkg, dev, c):
    """A row or two per group: the lanes stride over the contraction, 32768 products each.  (One
    running sum of equal products is off by 1e-4 and 3e-4.)"""
    import torch
    exact = torch.tensor(float(c) * LONG, device=dev, dtype=torch.float64)
    for E, rows in ((1, 4), (2, 6)):
        off = offsets(dev, [rows // E] * E)
        x, w = torch.ones(rows, LONG, device=dev), torch.full((E, 24, LONG), float(c), device=dev)
        assert_sums(pkg.grouped_matmul(x, w, off), exact.expand(rows, 24), "float32", FFMA)
    # The adapter's own product, A x, seen through B = 1 beside a projection of zeros.
    for T in (4, 70):
        y = pkg.lora_matmul(torch.ones(T, LONG, device=dev), torch.zeros(5, LONG, device=dev),
                            torch.full((1, 3, LONG), float(c), device=dev),
                            torch.ones(1, 5, 3, device=dev) / 4,
                            torch.zeros(T, dtype=torch.int32, device=dev), torch.ones(1, device=dev))
        assert_sums(y, (0.75 * exact).expand(T, 5), "float32", FFMA + 5 * 2.0 ** -24)


def test_fp32_grad_weight_of_many_rows(pkg, dev):
    """33 M rows in one expert.  (Sums of 512 and one running sum of those: off by 1.1e-4.)"""
    import torch
    rows, c = 1 << 25, 1 + 2.0 ** -12 - 2.0 ** -16
    x, dy = torch.full((rows, 1), c, device=dev), torch.ones(rows, 1, device=dev)
    dw = pkg.grouped_matmul_grad_weight(x, dy, offsets(dev, [rows]))
    exact = torch.full((1, 1, 1), c * rows, device=dev, dtype=torch.float64)
    assert_sums(dw, exact, "float32", FFMA)
