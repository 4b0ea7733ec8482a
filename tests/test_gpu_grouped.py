"""GPU parity of the expert products (grouped_matmul and its gradients) against float64.

Tolerance of one output, derived from the arithmetic: fp32 sums of c products lose at most
c * 2^-23 of the sum of magnitudes (one ulp, 2^-23, per added product covers rounding to
nearest and truncation alike, and the product's own rounding for fp32 operands adds 2^-24),
and the result is rounded once to the output type (half a step).  Both terms are counted with
the exact operands the device holds."""

import numpy as np
import pytest

from gpu_util import as_np, torch_dtype

pytestmark = pytest.mark.gpu

# Half a step of each type, relative to the value, and the smallest subnormal's half (an
# fp16 result below 2^-14 is rounded to a multiple of 2^-24).
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
FLOOR = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def bound(exact, mag, terms, dtype_name):
    acc = (terms + 1) * 2.0 ** -23 * mag
    return acc + HALF_STEP[dtype_name] * (np.abs(exact) + acc) + FLOOR[dtype_name]


def assert_close(got, exact, mag, terms, dtype_name):
    got = as_np(got)
    err, tol = np.abs(got - exact), bound(exact, mag, terms, dtype_name)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - tol), err.shape) if err.size else None
    assert (err <= tol).all(), f"{worst}: got {got[worst]}, exact {exact[worst]}, tol {tol[worst]}"


def offsets_of(counts, dev):
    import torch
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return torch.from_numpy(off).to(dev), off


def make(dev, counts, N, K, dtype_name, seed, extra_rows=0):
    import torch
    dt = torch_dtype(dtype_name)
    g = torch.Generator(device=dev).manual_seed(seed)
    R = int(sum(counts)) + extra_rows
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(dt)
    return rnd(R, K), rnd(len(counts), N, K) * 0.25, rnd(R, N)


# Rows per expert: empty ones first, last and in between, single rows, one row around every
# tile height, one expert with all rows.
COUNTS = {
    "one": [1],
    "single_rows": [1, 0, 1, 1, 0],
    "ragged": [0, 3, 17, 0, 64, 1, 130, 0],
    "edges": [15, 16, 17, 31, 33, 63, 65, 127, 128, 129],
    "tall": [0, 777, 0],
    "halves": [255, 256, 257, 511, 513, 2],
}
# (N, K): multiples of 8 around the tile sizes, below one tile, and odd sizes.
DIMS = [(8, 8), (40, 24), (128, 64), (136, 200), (264, 328), (33, 41), (130, 66), (1, 7)]


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("N,K", DIMS)
@pytest.mark.parametrize("counts", sorted(COUNTS))
def test_products_match_float64(pkg, orc, dev, dtype_name, N, K, counts):
    c = COUNTS[counts]
    x, w, dy = make(dev, c, N, K, dtype_name, seed=N * 1000 + K)
    off, hoff = offsets_of(c, dev)
    hx, hw, hdy = as_np(x), as_np(w), as_np(dy)
    y = pkg.grouped_matmul(x, w, off)
    assert_close(y, *orc.grouped_matmul(hx, hw, hoff), K, dtype_name)
    dx = pkg.grouped_matmul_grad_input(dy, w, off)
    assert_close(dx, *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, dtype_name)
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)
    assert_close(dw, *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(c), dtype_name)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("counts,N,K", [
    ([2, 0, 1, 5], 768, 2048), ([1] * 8 + [0] * 56, 768, 2048), ([300, 17, 1, 700], 512, 1024),
    ([9] * 30, 2048, 768), ([1024], 1032, 520), ([0, 0, 4], 4096, 4096), ([257] * 3, 520, 1032)])
def test_larger_products(pkg, orc, dev, dtype_name, counts, N, K):
    """Sizes that fill several tiles in every dimension, and long sums from few rows."""
    x, w, dy = make(dev, counts, N, K, dtype_name, seed=7)
    off, hoff = offsets_of(counts, dev)
    hx, hw, hdy = as_np(x), as_np(w), as_np(dy)
    assert_close(pkg.grouped_matmul(x, w, off), *orc.grouped_matmul(hx, hw, hoff), K, dtype_name)
    assert_close(pkg.grouped_matmul_grad_input(dy, w, off),
                 *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, dtype_name)
    assert_close(pkg.grouped_matmul_grad_weight(x, dy, off),
                 *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(counts), dtype_name)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("counts", [[3, 0, 30], [200, 300], [0, 0], [600, 1]])
def test_rows_behind_the_last_expert(pkg, orc, dev, dtype_name, counts):
    """Rows from offsets[E] on: never read (they hold NaN) and never written."""
    import torch
    N, K, extra = 72, 136, 37
    x, w, dy = make(dev, counts, N, K, dtype_name, seed=3, extra_rows=extra)
    used = sum(counts)
    x[used:], dy[used:] = float("nan"), float("nan")
    off, hoff = offsets_of(counts, dev)
    y = torch.full((used + extra, N), 7.0, device=dev, dtype=x.dtype)
    dx = torch.full((used + extra, K), 7.0, device=dev, dtype=x.dtype)
    pkg.grouped_matmul(x, w, off, out=y)
    pkg.grouped_matmul_grad_input(dy, w, off, out=dx)
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)
    assert (y[used:] == 7).all() and (dx[used:] == 7).all()
    hx, hw, hdy = as_np(x)[:used], as_np(w), as_np(dy)[:used]
    assert_close(y[:used], *orc.grouped_matmul(hx, hw, hoff), K, dtype_name)
    assert_close(dx[:used], *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, dtype_name)
    assert_close(dw, *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(counts), dtype_name)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("counts", [[5, 21, 3], [300, 260, 270]])
def test_non_finite_rows_stay_their_own(pkg, dev, dtype_name, counts):
    """NaN and infinities of one expert's rows and weights reach that expert's results only,
    and a row's NaN only that row."""
    import torch
    N, K = 136, 72
    x, w, dy = make(dev, counts, N, K, dtype_name, seed=5)
    off, hoff = offsets_of(counts, dev)
    clean = [pkg.grouped_matmul(x, w, off), pkg.grouped_matmul_grad_input(dy, w, off),
             pkg.grouped_matmul_grad_weight(x, dy, off)]
    lo, hi = int(hoff[1]), int(hoff[2])
    x[hi - 1], dy[hi - 1] = float("nan"), float("inf")
    y = pkg.grouped_matmul(x, w, off)
    dx = pkg.grouped_matmul_grad_input(dy, w, off)
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)
    rows = torch.arange(x.shape[0], device=dev) != hi - 1
    assert y[hi - 1].isnan().all() and not dx[hi - 1].isfinite().any()
    assert torch.equal(y[rows], clean[0][rows]) and torch.equal(dx[rows], clean[1][rows])
    assert torch.equal(dw[0], clean[2][0]) and torch.equal(dw[2], clean[2][2])
    assert dw[1].isnan().all()
    x2, w2, dy2 = make(dev, counts, N, K, dtype_name, seed=5)
    w2[1] = float("inf")
    y = pkg.grouped_matmul(x2, w2, off)
    dx = pkg.grouped_matmul_grad_input(dy2, w2, off)
    keep = torch.ones_like(rows)
    keep[lo:hi] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
def test_unaligned_buffers(pkg, orc, dev, dtype_name):
    """Contiguous tensors that start at an odd element of their storage."""
    import torch
    counts, N, K = [40, 7, 90], 64, 128
    x, w, dy = make(dev, counts, N, K, dtype_name, seed=11)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    off, hoff = offsets_of(counts, dev)
    hx, hw, hdy = as_np(x), as_np(w), as_np(dy)
    for sx, sw, sdy in [(shifted(x), w, dy), (x, shifted(w), shifted(dy))]:
        assert_close(pkg.grouped_matmul(sx, sw, off), *orc.grouped_matmul(hx, hw, hoff), K,
                     dtype_name)
        assert_close(pkg.grouped_matmul_grad_input(sdy, sw, off),
                     *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, dtype_name)
        assert_close(pkg.grouped_matmul_grad_weight(sx, sdy, off),
                     *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(counts), dtype_name)
    out = shifted(torch.zeros(sum(counts), N, device=dev, dtype=x.dtype))
    pkg.grouped_matmul(x, w, off, out=out)
    assert_close(out, *orc.grouped_matmul(hx, hw, hoff), K, dtype_name)


def test_offsets_out_of_range_are_clamped(pkg, orc, dev):
    """Offsets beyond the rows end at the last row, negative ones start at the first."""
    import torch
    x, w, dy = make(dev, [20, 30], 64, 64, "float16", seed=2)
    off = torch.tensor([-5, 20, 1 << 30], dtype=torch.int32, device=dev)
    y = pkg.grouped_matmul(x, w, off)
    assert_close(y, *orc.grouped_matmul(as_np(x), as_np(w), [0, 20, 50]), 64, "float16")
    dw = pkg.grouped_matmul_grad_weight(x, dy, off)
    assert_close(dw, *orc.grouped_matmul_grad_weight(as_np(x), as_np(dy), [0, 20, 50]), 30,
                 "float16")


@pytest.mark.parametrize("dtype_name,counts", [("float16", [300, 5, 0, 290]),
                                               ("bfloat16", [2, 1, 0, 3]),
                                               ("float32", [300, 5, 0, 290])])
def test_repeated_captured_and_streamed_calls(pkg, dev, dtype_name, counts):
    """The same bits from a second call, from two captured graphs replayed on new inputs, and
    from calls on two other streams at once."""
    import torch
    x, w, dy = make(dev, counts, 264, 520, dtype_name, seed=9)
    off, _ = offsets_of(counts, dev)

    def all3(stream=None):
        return (pkg.grouped_matmul(x, w, off, stream=stream),
                pkg.grouped_matmul_grad_input(dy, w, off, stream=stream),
                pkg.grouped_matmul_grad_weight(x, dy, off, stream=stream))

    first = all3()
    assert all(torch.equal(a, b) for a, b in zip(first, all3()))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = all3()
        graphs.append((g, out))
    x2, _, dy2 = make(dev, counts, 264, 520, dtype_name, seed=10)
    x0, dy0 = x.clone(), dy.clone()
    x.copy_(x2), dy.copy_(dy2)
    want = all3()
    for g, out in graphs + graphs:
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))
    x.copy_(x0), dy.copy_(dy0)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [all3(s) for s in (s1, s2, s1.cuda_stream, s2)]
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(first, o))


def test_gradients_match_differences(pkg, dev):
    """f(x, w) = sum(dy * y) is linear in x and in w, so central differences of the forward
    product along a direction equal <dx, d> and <dw, d> up to rounding: each side sums R N
    (or R K, E N K) fp32-rounded terms, bounded by its sum of magnitudes."""
    import torch
    counts, N, K = [50, 0, 33, 9], 96, 72
    x, w, dy = make(dev, counts, N, K, "float32", seed=21)
    dxd, dwd, _ = make(dev, counts, N, K, "float32", seed=22)
    off, _ = offsets_of(counts, dev)
    f = lambda xx, ww: (dy.double() * pkg.grouped_matmul(xx, ww, off).double()).sum().item()
    dx = pkg.grouped_matmul_grad_input(dy, w, off).double()
    dw = pkg.grouped_matmul_grad_weight(x, dy, off).double()
    h = 0.5  # exact in fp32; the function is linear, so the step need not be small
    mag = (dy.abs().double() * pkg.grouped_matmul(x.abs() + dxd.abs(), w.abs() + dwd.abs(),
                                                  off).double()).sum().item()
    tol = 4 * (max(N, K, max(counts)) + 2) * 2.0 ** -23 * mag
    assert abs((f(x + h * dxd, w) - f(x - h * dxd, w)) / (2 * h) -
               (dx * dxd.double()).sum().item()) <= tol
    assert abs((f(x, w + h * dwd) - f(x, w - h * dwd)) / (2 * h) -
               (dw * dwd.double()).sum().item()) <= tol
    assert tol < 1e-2 * abs((dx * dx).sum().item())  # the bound says something


def test_element_offsets_past_32_bits(pkg, dev):
    """2.3 G output elements: the last expert's rows lie past 2^31 elements."""
    import torch
    counts, N, K = [500_000, 60_000, 13], 4096, 64
    R = sum(counts)
    dt = torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(R, K, device=dev, generator=g).to(dt)
    w = torch.randn(3, N, K, device=dev, generator=g).to(dt)
    off, hoff = offsets_of(counts, dev)
    y = pkg.grouped_matmul(x, w, off)
    dx = pkg.grouped_matmul_grad_input(y, w, off)
    dw = pkg.grouped_matmul_grad_weight(x, y, off)
    for p in (0, 499_999, 500_000, 524_287, 524_288, R - 13, R - 1):
        e = int(np.searchsorted(hoff, p, side="right")) - 1
        ref = w[e].double() @ x[p].double()
        mag = w[e].double().abs() @ x[p].double().abs()
        tol = 2.0 ** -8 * ref.abs() + 2 * K * 2.0 ** -23 * mag
        assert ((y[p].double() - ref).abs() <= tol).all()
        ref = w[e].double().t() @ y[p].double()
        mag = w[e].double().abs().t() @ y[p].double().abs()
        tol = 2.0 ** -8 * ref.abs() + 2 * N * 2.0 ** -23 * mag
        assert ((dx[p].double() - ref).abs() <= tol).all()
    last = slice(R - 13, R)
    ref = y[last].double().t() @ x[last].double()
    mag = y[last].double().abs().t() @ x[last].double().abs()
    assert ((dw[2].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 28 * 2.0 ** -23 * mag).all()


def test_wrapper_refusals(pkg, dev):
    import torch
    x, w, dy = make(dev, [4, 4], 16, 24, "float16", seed=0)
    off, _ = offsets_of([4, 4], dev)
    with pytest.raises(TypeError, match="weights"):
        pkg.grouped_matmul(x, w.float(), off)
    with pytest.raises(TypeError, match="expert_offsets"):
        pkg.grouped_matmul(x, w, off.long())
    with pytest.raises(ValueError, match="shape"):
        pkg.grouped_matmul(x, w, off[:2].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        pkg.grouped_matmul(x.t(), w.transpose(1, 2), off)
    with pytest.raises(ValueError, match="shape"):
        pkg.grouped_matmul(x[:, :16].contiguous(), w, off)
    with pytest.raises(ValueError, match="out"):
        pkg.grouped_matmul(x, w, off, out=torch.empty(8, 24, device=dev, dtype=x.dtype))
    with pytest.raises(ValueError, match="shape"):
        pkg.grouped_matmul_grad_weight(x, dy[:4].contiguous(), off)
    with pytest.raises(ValueError, match="contiguous tensor on"):
        pkg.grouped_matmul(x, w, off.cpu())


def test_no_rows(pkg, dev):
    import torch
    x = torch.empty(0, 24, device=dev, dtype=torch.float16)
    w = torch.randn(3, 16, 24, device=dev).half()
    off = torch.zeros(4, dtype=torch.int32, device=dev)
    assert pkg.grouped_matmul(x, w, off).shape == (0, 16)
    dy = torch.empty(0, 16, device=dev, dtype=torch.float16)
    assert pkg.grouped_matmul_grad_input(dy, w, off).shape == (0, 24)
    out = torch.full((3, 16, 24), 5.0, device=dev, dtype=torch.float16)
    pkg.grouped_matmul_grad_weight(x, dy, off, out=out)
    assert not out.any()


# Long fp32 contractions.  Every product is c = 1 + 2^-13 - 2^-16 (times a power of two per row),
# chosen so that one running sum of 4096 or more of them rounds the same way at every step: off
# by 4.7e-5 to 9.2e-5 of the sum for 1 to 4 such sums, computed in fp32.  Sums of 512 and then a
# sum of those lose at most one half step per addition on the way of a product:
# 512 + 16384 / 512 additions, four more where the contraction is split.
LONG = 16384


def long_bound(exact):
    return np.abs(exact) * (512 + LONG // 512 + 4) * 2.0 ** -24


@pytest.mark.parametrize("rows,feat,E", [(4, 24, 1), (24, 40, 2), (70, 72, 1), (768, 896, 1)])
def test_fp32_long_sums(pkg, dev, rows, feat, E):
    import torch
    c = 1 + 2.0 ** -13 - 2.0 ** -16
    off, _ = offsets_of([rows // E] * E, dev)
    scale = torch.tensor([2.0 ** (i % 5 - 2) for i in range(rows)], device=dev)
    a = scale[:, None].expand(rows, LONG).contiguous()
    exact = (as_np(scale) * c * LONG)[:, None]
    got = as_np(pkg.grouped_matmul(a, torch.full((E, feat, LONG), c, device=dev), off))
    assert (np.abs(got - exact) <= long_bound(exact)).all()
    got = as_np(pkg.grouped_matmul_grad_input(a, torch.full((E, LONG, feat), c, device=dev), off))
    assert (np.abs(got - exact) <= long_bound(exact)).all()
    # The weights' gradient sums over rows: an expert with all of them, beside an empty one.
    off, _ = offsets_of([LONG, 0], dev)
    dy = scale[None, :].expand(LONG, rows).contiguous()
    got = as_np(pkg.grouped_matmul_grad_weight(torch.full((LONG, feat), c, device=dev), dy, off))
    assert (np.abs(got[0] - exact) <= long_bound(exact)).all()
    assert (got[1] == 0).all()


def test_output_over_an_input_is_refused(pkg, dev):
    import torch
    x = torch.zeros(8, 16, dtype=torch.float16, device=dev)
    w = torch.zeros(1, 16, 16, dtype=torch.float16, device=dev)
    off, _ = offsets_of([8], dev)
    for call in (pkg.grouped_matmul, pkg.grouped_matmul_grad_input):
        with pytest.raises(pkg.MoeB200Error, match="overlap"):
            call(x, w, off, out=x)
    both = torch.zeros(2, 8, 16, dtype=torch.float16, device=dev)
    call(both[0], w, off, out=both[1])  # neighbours do not overlap


# One process: its first call of every kernel happens inside a capture.
FIRST_CALL_CAPTURED = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from __graft_entry__ import load_package
pkg = load_package()
dev = torch.device("cuda", 0)
off = torch.tensor([0, 300, 300, 600], dtype=torch.int32, device=dev)
ids = torch.arange(600, dtype=torch.int32, device=dev) % 5 - 1
sc = torch.ones(4, device=dev)
calls = []
for dt in (torch.float32, torch.bfloat16):
    t = lambda *s: torch.randn(*s, device=dev).to(dt)
    x, w, dy, a, b = t(600, 64), t(3, 128, 64), t(600, 128), t(4, 16, 64), t(4, 128, 16)
    calls += [lambda x=x, w=w: pkg.grouped_matmul(x, w, off),
              lambda dy=dy, w=w: pkg.grouped_matmul_grad_input(dy, w, off),
              lambda x=x, dy=dy: pkg.grouped_matmul_grad_weight(x, dy, off),
              lambda x=x, w=w, a=a, b=b: pkg.lora_matmul(x, w[0], a, b, ids, sc),
              lambda x=x, w=w, a=a, b=b: pkg.lora_matmul(x[:3], w[0], a, b, ids[:3], sc)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = [c() for c in calls]
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(o, c()) for o, c in zip(out, calls))
"""


def test_first_call_may_be_captured(dev):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, root], cwd=root, timeout=300,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


def test_traced_calls(pkg, dev, monkeypatch):
    """With MOE_B200_TRACE_SYNC every call waits and looks for a device error: same bits."""
    import torch
    x, w, dy = make(dev, [300, 5, 0], 72, 64, "float16", seed=3)
    off, _ = offsets_of([300, 5, 0], dev)
    ids = torch.arange(x.shape[0], dtype=torch.int32, device=dev) % 3 - 1
    a = torch.randn(2, 8, 64, device=dev).half()
    b = torch.randn(2, 72, 8, device=dev).half()
    sc = torch.ones(2, device=dev)

    def all4():
        return (pkg.grouped_matmul(x, w, off), pkg.grouped_matmul_grad_input(dy, w, off),
                pkg.grouped_matmul_grad_weight(x, dy, off),
                pkg.lora_matmul(x, w[0], a, b, ids, sc),
                pkg.lora_matmul(x[:4], w[0], a, b, ids[:4], sc))

    want = all4()
    monkeypatch.setenv("MOE_B200_TRACE_SYNC", "1")
    assert all(torch.equal(p, q) for p, q in zip(want, all4()))
