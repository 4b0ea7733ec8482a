"""Waits of the expert products and the adapter projection that run out, without a fault: with
the test hook MOE_B200_TEST_STALL=1 the tensor-core kernels' producers issue no loads, so every
role waits for barriers that never complete, gives up after 2 s each, frees its tensor memory and
leaves.  The caller is told: by the next call on the device, by take_device_error(), or under
MOE_B200_TRACE_SYNC by the call itself."""

import time

import pytest

pytestmark = pytest.mark.gpu


def calls(pkg, dev):
    """One call for each kernel."""
    import torch
    g = torch.Generator(device=dev).manual_seed(0)
    t = lambda *s: torch.randn(*s, device=dev, generator=g).bfloat16()
    off = lambda *o: torch.tensor(o, dtype=torch.int32, device=dev)
    x, w = t(2048, 64), t(1, 2048, 64)
    a, b = t(3, 16, 64), t(3, 2048, 16)
    ids, sc = torch.arange(2048, dtype=torch.int32, device=dev) % 4 - 1, torch.ones(3, device=dev)
    run = torch.arange(2048, dtype=torch.int32, device=dev) // 700
    lora = lambda n, i: pkg.lora_matmul(x[:n], w[0], a, b, i[:n].contiguous(), sc)
    return dict(
        pair=lambda: pkg.grouped_matmul(x, w, off(0, 2048)),
        pair_grad_weight=lambda: pkg.grouped_matmul_grad_weight(x[:100], x[100:200], off(0, 7, 7, 99)),
        streaming=lambda: pkg.grouped_matmul(x[:3], w, off(0, 3)),
        lora_one_launch=lambda: lora(3, ids), lora_streaming=lambda: lora(40, ids),
        lora_mixed=lambda: lora(2048, ids), lora_runs=lambda: lora(2048, run))


@pytest.mark.parametrize("name", ["pair", "pair_grad_weight", "streaming", "lora_one_launch",
                                  "lora_streaming", "lora_mixed", "lora_runs"])
def test_next_call_reports_a_wait_that_ran_out(pkg, dev, monkeypatch, name):
    import torch
    call = calls(pkg, dev)[name]
    want = call()
    torch.cuda.synchronize()
    t0 = time.time()
    monkeypatch.setenv("MOE_B200_TEST_STALL", "1")
    call()
    monkeypatch.delenv("MOE_B200_TEST_STALL")
    torch.cuda.synchronize()
    assert time.time() - t0 < 40
    with pytest.raises(pkg.EPFail, match="earlier .*device error code"):
        call()
    assert torch.equal(call(), want)
    assert pkg.take_device_error() == 0


def test_error_can_be_asked_for(pkg, dev, monkeypatch):
    import torch
    call = calls(pkg, dev)["streaming"]
    want = call()
    monkeypatch.setenv("MOE_B200_TEST_STALL", "1")
    call()
    monkeypatch.delenv("MOE_B200_TEST_STALL")
    torch.cuda.synchronize()
    assert pkg.take_device_error() in (1, 2, 3)
    assert pkg.take_device_error() == 0
    assert torch.equal(call(), want)


def test_traced_call_reports_its_own_error(pkg, dev, monkeypatch):
    """... and leaves none for the next call."""
    import torch
    call = calls(pkg, dev)["streaming"]
    want = call()
    monkeypatch.setenv("MOE_B200_TEST_STALL", "1")
    monkeypatch.setenv("MOE_B200_TRACE_SYNC", "1")
    with pytest.raises(pkg.EPFail, match="grouped_matmul: device error code"):
        call()
    monkeypatch.delenv("MOE_B200_TEST_STALL")
    assert pkg.take_device_error() == 0
    assert torch.equal(call(), want)


def test_traced_call_may_be_captured(pkg, dev, monkeypatch):
    """Nothing has run at the end of a captured call: it neither waits nor spoils the capture."""
    import torch
    call = calls(pkg, dev)["lora_streaming"]
    x = torch.ones(2, 8, device=dev)
    w = torch.ones(1, 8, 8, device=dev)
    off = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    want = pkg.grouped_matmul(x, w, off)
    monkeypatch.setenv("MOE_B200_TRACE_SYNC", "1")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = pkg.grouped_matmul(x, w, off)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and call() is not None


def test_replays_of_a_call_captured_while_traced_report_their_errors(pkg, dev, monkeypatch):
    """A replay is waited for by nobody, so the next call has to tell."""
    import torch
    call = calls(pkg, dev)["streaming"]
    want = call()
    monkeypatch.setenv("MOE_B200_TEST_STALL", "1")
    monkeypatch.setenv("MOE_B200_TRACE_SYNC", "1")
    g = torch.cuda.CUDAGraph()
    off = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    x, w = torch.ones(3, 64, device=dev).half(), torch.ones(1, 64, 64, device=dev).half()
    with torch.cuda.graph(g):
        pkg.grouped_matmul(x, w, off)
    monkeypatch.delenv("MOE_B200_TEST_STALL")
    monkeypatch.delenv("MOE_B200_TRACE_SYNC")
    g.replay()
    torch.cuda.synchronize()
    with pytest.raises(pkg.EPFail, match="earlier .*device error code"):
        call()
    assert torch.equal(call(), want)
