"""GPU parity of the adapter projection (lora_matmul) against float64.

Tolerance of one output: the shared product as in test_gpu_grouped.py, (k + r + 2) * 2^-23 of
its sum of magnitudes; the adapter term loses (k + 1) * 2^-23 of its magnitude in the fp32
intermediate, 2^-15 where that intermediate enters the tensor cores as the sum of two 16-bit
parts (each part rounds by at most 2^-8 of what it represents in bf16, so two parts leave
2^-16, doubled here for the products of the rounding errors), and (r + 4) * 2^-23 in its own
sum and scaling; the result is rounded once to the output type."""

import numpy as np
import pytest

from gpu_util import as_np, to_dev, torch_dtype
from test_gpu_grouped import FLOOR, HALF_STEP

pytestmark = pytest.mark.gpu


def assert_lora(got, exact, mag, mag_l, k, r, dtype_name):
    got = as_np(got)
    acc = (k + r + 2) * 2.0 ** -23 * mag
    split = 0.0 if dtype_name == "float32" else 2.0 ** -15
    acc = acc + ((k + r + 6) * 2.0 ** -23 + split) * mag_l
    tol = acc + HALF_STEP[dtype_name] * (np.abs(exact) + acc) + FLOOR[dtype_name]
    err = np.abs(got - exact)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), f"{worst}: got {got[worst]}, exact {exact[worst]}, tol {tol[worst]}"


def make(dev, T, N, K, r, L, dtype_name, ids, seed=0):
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = torch_dtype(dtype_name)
    rnd = lambda s, *sh: (torch.randn(*sh, device=dev, generator=g) * s).to(dt)
    d = dict(x=rnd(1.0, T, K), weight=rnd(K ** -0.5, N, K), lora_a=rnd(K ** -0.5, L, r, K),
             lora_b=rnd(0.5, L, N, r), adapter_ids=torch.as_tensor(ids, dtype=torch.int32).to(dev),
             scales=torch.rand(L, device=dev, generator=g) * 2 - 0.5)
    return d


def oracle(orc, d):
    return orc.lora_matmul(as_np(d["x"]), as_np(d["weight"]), as_np(d["lora_a"]),
                           as_np(d["lora_b"]), d["adapter_ids"].cpu().numpy(),
                           as_np(d["scales"]))


def ids_of(kind, T, L, rng):
    if kind == "none":
        return np.full(T, -1)
    if kind == "one":
        return np.full(T, L - 1)
    if kind == "mixed":
        return rng.integers(-1, L, T)
    if kind == "foreign":  # ids outside [0, L) mean no adapter
        return rng.choice([-1, -7, L, 2 ** 31 - 1, 0], T)
    runs = np.repeat(rng.integers(-1, L, T // 37 + 1), 37)[:T]  # prompts of 37 rows
    return runs


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("T,N,K,r,L", [
    (1, 64, 64, 8, 1), (1, 264, 520, 16, 3), (7, 72, 136, 8, 4), (16, 128, 256, 32, 5),
    (33, 136, 200, 16, 9), (65, 264, 328, 64, 3), (130, 520, 264, 24, 40), (257, 128, 128, 128, 2),
    (600, 264, 136, 16, 7), (5, 33, 41, 3, 2), (70, 130, 66, 5, 6), (300, 64, 72, 256, 3),
    (9, 8, 8, 1, 2), (1, 136, 72, 128, 2), (2, 1032, 264, 64, 3), (3, 520, 136, 40, 2),
    (8, 264, 2056, 16, 5), (8, 64, 64, 8, 3), (4, 4104, 520, 24, 6)])
@pytest.mark.parametrize("kind", ["none", "one", "mixed", "foreign", "runs"])
def test_lora_matches_float64(pkg, orc, dev, dtype_name, T, N, K, r, L, kind):
    rng = np.random.default_rng(T * 7 + r)
    d = make(dev, T, N, K, r, L, dtype_name, ids_of(kind, T, L, rng), seed=T)
    y = pkg.lora_matmul(**d)
    assert_lora(y, *oracle(orc, d), K, r, dtype_name)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16"])
@pytest.mark.parametrize("T,N,K,r,L,kind", [
    (1, 4096, 4096, 16, 8, "one"), (64, 1024, 4096, 16, 32, "mixed"), (64, 1032, 2056, 64, 64, "mixed"),
    (300, 1024, 2048, 16, 6, "runs"), (1100, 2048, 1024, 64, 5, "runs"), (1025, 520, 1032, 8, 100, "mixed"),
    (1500, 2568, 520, 16, 7, "runs"), (1300, 2560, 264, 24, 9, "mixed"), (3001, 1544, 136, 136, 4, "runs"),
    (1281, 2816, 72, 8, 3, "foreign")])
def test_larger_lora(pkg, orc, dev, dtype_name, T, N, K, r, L, kind):
    rng = np.random.default_rng(3)
    d = make(dev, T, N, K, r, L, dtype_name, ids_of(kind, T, L, rng), seed=1)
    assert_lora(pkg.lora_matmul(**d), *oracle(orc, d), K, r, dtype_name)


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("T", [6, 70, 700])
def test_other_adapters_do_not_reach_a_row(pkg, dev, dtype_name, T):
    """An adapter full of NaN and infinities, and a row of NaN, change no other row."""
    import torch
    L = 4
    ids = np.arange(T) % L
    ids[::5] = -1
    d = make(dev, T, 136, 264, 16, L, dtype_name, ids, seed=4)
    clean = pkg.lora_matmul(**d)
    d["lora_a"][1] = float("nan")
    d["lora_b"][1] = float("inf")
    d["lora_b"][3, :, 2] = float("inf")
    d["scales"][1] = float("nan")
    y = pkg.lora_matmul(**d)
    mine = torch.as_tensor((ids != 1) & (ids != 3), device=dev)
    assert torch.equal(y[mine], clean[mine])
    hit = torch.as_tensor(ids == 1, device=dev)
    assert not y[hit].isfinite().any()
    d = make(dev, T, 136, 264, 16, L, dtype_name, ids, seed=4)
    d["x"][T // 2] = float("nan")
    y = pkg.lora_matmul(**d)
    rows = torch.arange(T, device=dev) != T // 2
    assert y[T // 2].isnan().all() and torch.equal(y[rows], clean[rows])


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("T", [3, 300])
def test_intermediate_beyond_the_16_bit_range(pkg, orc, dev, dtype_name, T):
    """A_a x up to about 1e6 (past fp16) scaled back by small B and scales."""
    d = make(dev, T, 128, 512, 16, 2, dtype_name, np.arange(T) % 2, seed=8)
    d["lora_a"] *= 32768.0
    d["lora_b"] *= 2.0 ** -10
    d["scales"] *= 2.0 ** -6
    assert_lora(pkg.lora_matmul(**d), *oracle(orc, d), 512, 16, dtype_name)


@pytest.mark.parametrize("dtype_name,T", [("float16", 2), ("bfloat16", 100), ("bfloat16", 700),
                                          ("float32", 50)])
def test_repeated_captured_and_streamed_calls(pkg, dev, dtype_name, T):
    import torch
    ids = np.arange(T) % 5 - 1
    d = make(dev, T, 264, 520, 16, 4, dtype_name, ids, seed=9)
    first = pkg.lora_matmul(**d)
    assert torch.equal(first, pkg.lora_matmul(**d))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, pkg.lora_matmul(**d)))
    d2 = make(dev, T, 264, 520, 16, 4, dtype_name, ids[::-1].copy(), seed=10)
    keep = {n: d[n].clone() for n in ("x", "adapter_ids")}
    for n in keep:
        d[n].copy_(d2[n])
    want = pkg.lora_matmul(**d)
    for g, out in graphs + graphs:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, out)
    for n, t in keep.items():
        d[n].copy_(t)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [pkg.lora_matmul(**d, stream=s) for s in (s1, s2, s1, s2.cuda_stream)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in got)


def test_unaligned_buffers(pkg, orc, dev):
    import torch
    d = make(dev, 40, 64, 128, 8, 3, "bfloat16", np.arange(40) % 4 - 1, seed=2)
    ref = oracle(orc, d)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    for name in ("x", "weight", "lora_a", "lora_b"):
        e = dict(d, **{name: shifted(d[name])})
        assert_lora(pkg.lora_matmul(**e), *ref, 128, 8, "bfloat16")
    out = shifted(torch.zeros(40, 64, device=dev, dtype=torch.bfloat16))
    pkg.lora_matmul(**d, out=out)
    assert_lora(out, *ref, 128, 8, "bfloat16")


def test_wrapper_refusals(pkg, dev):
    import torch
    d = make(dev, 8, 32, 64, 8, 2, "float16", np.zeros(8), seed=2)
    with pytest.raises(TypeError, match="scales"):
        pkg.lora_matmul(**dict(d, scales=d["scales"].half()))
    with pytest.raises(TypeError, match="adapter_ids"):
        pkg.lora_matmul(**dict(d, adapter_ids=d["adapter_ids"].long()))
    with pytest.raises(ValueError, match="lora_b"):
        pkg.lora_matmul(**dict(d, lora_b=d["lora_b"][:, :, :4].contiguous()))
    with pytest.raises(ValueError, match="contiguous"):
        pkg.lora_matmul(**dict(d, weight=d["weight"].t().contiguous().t()))
    with pytest.raises(pkg.InvalidArgument, match="rank"):
        pkg.lora_matmul(**dict(d, lora_a=torch.zeros(2, 257, 64, device=dev, dtype=torch.float16),
                               lora_b=torch.zeros(2, 32, 257, device=dev, dtype=torch.float16)))
    assert pkg.lora_matmul(**dict(d, x=d["x"][:0], adapter_ids=d["adapter_ids"][:0])).shape == (0, 32)


def test_adapted_projection_feeds_an_expert_layer(pkg, orc, dev):
    """The operators as a block uses them: an adapted output projection, the residual and the
    router, the dispatch plan, both expert products around the activation and the combine --
    against the layer kernel on the same rows -- and the layer's weight and input gradients
    against float64."""
    import torch
    T, H, I, E, k, L, r = 150, 256, 384, 8, 2, 3, 16
    dt = torch.bfloat16
    ids = np.repeat([0, 1, -1, 2], 40)[:T]
    d = make(dev, T, H, H, r, L, "bfloat16", ids, seed=31)
    rng = np.random.default_rng(32)
    t = lambda a, dtype=dt: to_dev(a.astype(np.float32), dev, dtype)
    skip = t(rng.standard_normal((T, H)))
    gamma = t(1 + 0.1 * rng.standard_normal(H), torch.float32)
    wr = t(0.05 * rng.standard_normal((E, H)))
    fc1, fc3 = (t(0.05 * rng.standard_normal((E, I, H))) for _ in range(2))
    fc2 = t(0.05 * rng.standard_normal((E, H, I)))

    h = pkg.lora_matmul(**d)
    normed, logits, _ = pkg.norm_router(h, gamma, 1e-5, wr, skip=skip)
    idx, weight = pkg.route(logits, k, 1)
    off, pos, src = pkg.permute(idx, E)
    xp = normed[(src // k).long()]
    g, u = pkg.grouped_matmul(xp, fc1, off), pkg.grouped_matmul(xp, fc3, off)
    act = (torch.nn.functional.silu(g.float()) * u.float()).to(dt)
    y = pkg.grouped_matmul(act, fc2, off)
    out = pkg.ep_combine(y, pos, weight, torch.empty_like(normed))
    op = pkg.MoE(activation_type="silu", k=k, normalize_routing_weights=1)
    layer = op([normed, logits, fc1, None, fc2, None, fc3, None])
    op.release()
    torch.cuda.synchronize()
    # The layer kernel rounds the activation once where the composition rounds g and u too:
    # three roundings of half a step in the activation against one, seen through fc2's sum.
    a64 = as_np(act)
    _, mag = orc.grouped_matmul(a64, as_np(fc2), off.cpu().numpy())
    hm = np.zeros((T, H))
    np.add.at(hm, (src.cpu().numpy() // k), mag * as_np(weight).reshape(-1)[src.cpu().numpy()][:, None])
    tol = 8 * 2.0 ** -8 * hm + 4 * 2.0 ** -8 * np.abs(as_np(layer)) + 1e-6
    assert (np.abs(as_np(out) - as_np(layer)) <= tol).all()

    # One backward step of the experts: d out -> dy -> d act, d fc2 -> (silu, product) -> d xp.
    gout = t(rng.standard_normal((T, H)))
    w_of = weight.reshape(-1)[src.long()]
    dy = (gout.float()[(src // k).long()] * w_of[:, None]).to(dt)
    hoff = off.cpu().numpy()
    from test_gpu_grouped import assert_close
    dact = pkg.grouped_matmul_grad_input(dy, fc2, off)
    assert_close(dact, *orc.grouped_matmul_grad_input(as_np(dy), as_np(fc2), hoff), H, "bfloat16")
    dfc2 = pkg.grouped_matmul_grad_weight(act, dy, off)
    counts = int(np.diff(hoff).max())
    assert_close(dfc2, *orc.grouped_matmul_grad_weight(as_np(act), as_np(dy), hoff), counts,
                 "bfloat16")
    sg = torch.sigmoid(g.float())
    dg = (dact.float() * u.float() * (sg * (1 + g.float() * (1 - sg)))).to(dt)
    du = (dact.float() * torch.nn.functional.silu(g.float())).to(dt)
    dxp = pkg.grouped_matmul_grad_input(dg, fc1, off).float() + \
        pkg.grouped_matmul_grad_input(du, fc3, off).float()
    e1, m1 = orc.grouped_matmul_grad_input(as_np(dg), as_np(fc1), hoff)
    e3, m3 = orc.grouped_matmul_grad_input(as_np(du), as_np(fc3), hoff)
    tol = 2.0 ** -8 * (np.abs(e1) + np.abs(e3)) + (I + 4) * 2.0 ** -22 * (m1 + m3)
    assert (np.abs(as_np(dxp) - (e1 + e3)) <= tol).all()
    dfc1 = pkg.grouped_matmul_grad_weight(xp, dg, off)
    assert_close(dfc1, *orc.grouped_matmul_grad_weight(as_np(xp), as_np(dg), hoff), counts,
                 "bfloat16")
