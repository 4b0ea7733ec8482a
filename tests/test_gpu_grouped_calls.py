"""The expert products and the adapter projection in the settings that a program calls them in."""

import os
import subprocess
import sys

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


# One process, since the switch is read once: captures a chain of calls and counts the graph's
# programmatic edges (a kernel that may start while the one in front drains).
EDGES = """
import ctypes, sys, torch
sys.path.insert(0, sys.argv[1])
from __graft_entry__ import load_package
pkg = load_package()
dev = torch.device("cuda", 0)
off = torch.tensor([0, 30, 30, 60], dtype=torch.int32, device=dev)
ids = torch.arange(60, dtype=torch.int32, device=dev) % 3
sc = torch.ones(3, device=dev)
calls = []
for dt, rank in ((torch.float32, 5), (torch.bfloat16, 16)):
    t = lambda *s: torch.randn(*s, device=dev).to(dt)
    x, w, dy, a, b = t(60, 64), t(3, 128, 64), t(60, 128), t(3, rank, 64), t(3, 128, rank)
    calls += [lambda x=x, w=w: pkg.grouped_matmul(x, w, off),
              lambda dy=dy, w=w: pkg.grouped_matmul_grad_input(dy, w, off),
              lambda x=x, dy=dy: pkg.grouped_matmul_grad_weight(x, dy, off),
              lambda x=x, w=w, a=a, b=b: pkg.lora_matmul(x, w[0], a, b, ids, sc),
              lambda x=x, w=w, a=a, b=b: pkg.lora_matmul(x[:3], w[0], a, b, ids[:3], sc)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(g):
    out = [c() for c in calls]
drv = ctypes.CDLL("libcuda.so.1")
raw, n = ctypes.c_void_p(g.raw_cuda_graph()), ctypes.c_size_t(0)
assert drv.cuGraphGetEdges_v2(raw, None, None, None, ctypes.byref(n)) == 0
nodes, data = (ctypes.c_void_p * n.value)(), (ctypes.c_ubyte * (8 * n.value))()
assert drv.cuGraphGetEdges_v2(raw, nodes, (ctypes.c_void_p * n.value)(), data, ctypes.byref(n)) == 0
print("edges", n.value, "programmatic", sum(data[8 * i + 2] == 1 for i in range(n.value)))
g.instantiate()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(o, c()) for o, c in zip(out, calls))
"""


@pytest.mark.parametrize("switch", ["0", "1"])
def test_overlapped_launches_can_be_turned_off(dev, switch):
    """MOE_B200_PDL=0 holds for these calls too, with the same bits."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", EDGES, root], cwd=root, timeout=300,
                          env=dict(os.environ, MOE_B200_PDL=switch), capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
    edges, programmatic = (int(w) for w in done.stdout.split()[1::2])
    assert edges >= 10 and (programmatic == 0 if switch == "0" else programmatic >= 8)


LOADS = {
    "all rows in one": [0] * 100 + [700] + [0] * 155,
    "one row each": [1] * 256,
    "a few each": [(7 * e) % 10 for e in range(256)],
    "last only": [0] * 255 + [3],
    "tiles of each": [90 - e % 5 for e in range(256)],
}


@pytest.mark.parametrize("dtype_name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("load", sorted(LOADS))
def test_as_many_experts_as_there_may_be(pkg, orc, dev, dtype_name, load):
    """256 experts: every group table is full, and the rules that choose a kernel see the mean."""
    counts, N, K = LOADS[load], 72, 136
    x, w, dy = make(dev, counts, N, K, dtype_name, seed=13)
    off, hoff = offsets_of(counts, dev)
    hx, hw, hdy = as_np(x), as_np(w), as_np(dy)
    assert_close(pkg.grouped_matmul(x, w, off), *orc.grouped_matmul(hx, hw, hoff), K, dtype_name)
    assert_close(pkg.grouped_matmul_grad_input(dy, w, off),
                 *orc.grouped_matmul_grad_input(hdy, hw, hoff), N, dtype_name)
    assert_close(pkg.grouped_matmul_grad_weight(x, dy, off),
                 *orc.grouped_matmul_grad_weight(hx, hdy, hoff), max(counts), dtype_name)


def test_calls_from_several_threads(pkg, dev):
    """Threads with a stream each, at once: the bits of a single thread."""
    import threading
    import torch
    x, w, dy = make(dev, [300, 0, 5, 60], 264, 520, "bfloat16", seed=14)
    off, _ = offsets_of([300, 0, 5, 60], dev)
    ids = torch.arange(365, dtype=torch.int32, device=dev) % 4 - 1
    a, b, sc = torch.randn(3, 16, 520, device=dev).bfloat16(), \
        torch.randn(3, 264, 16, device=dev).bfloat16(), torch.rand(3, device=dev)

    def all4(n):
        return [pkg.grouped_matmul(x, w, off), pkg.grouped_matmul_grad_input(dy, w, off),
                pkg.grouped_matmul_grad_weight(x, dy, off),
                pkg.lora_matmul(x[:n], w[0], a, b, ids[:n], sc)]

    rows = (3, 60, 365, 20)
    want = [all4(n) for n in rows]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(20):
                    out = all4(rows[i])
                torch.cuda.current_stream().synchronize()
            got[i] = out
        except Exception as e:  # noqa: BLE001 -- shown below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(rows))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert all(torch.equal(p, q) for i in got for p, q in zip(want[i], got[i])) and len(got) == 4
