"""A workspace made inside a capture is that call's alone: only the graph's replays zero it, so a call outside that took
it for the device's shared one would find whatever the memory held."""
import pytest
import torch

from conftest import randn_f16
from whisper_blaze_b200 import _lib, ops

DEV = torch.device("cuda", 0)


def test_the_shared_one_stays_what_it_was(monkeypatch):
    monkeypatch.setattr(ops, "_zeros", lambda nbytes, device: torch.zeros(nbytes, dtype=torch.uint8))
    monkeypatch.setattr(ops, "_SPLITK_WS", {})
    monkeypatch.setattr(ops, "_SPLITK_OUTGROWN", {})
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    for capturing, nbytes in ((True, 512), (False, 256), (True, 1024), (True, 256)):
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        before = ops._SPLITK_WS.get(DEV)
        ws = ops.splitk_workspace(DEV, nbytes)
        assert ws.numel() >= nbytes and int(ws.count_nonzero()) == 0
        if capturing:
            assert ops._SPLITK_WS.get(DEV) is before
            assert (ws is before) is (before is not None and before.numel() >= nbytes)
        else:
            assert ops._SPLITK_WS[DEV] is ws
    assert not ops._SPLITK_OUTGROWN


@pytest.mark.gpu
def test_a_linear_after_a_capture_that_came_first(cuda_device, monkeypatch):
    x = randn_f16((64, 1280), 90).to(cuda_device)
    w, scale = ops.quantise(randn_f16((1280, 1280), 91, std=0.02).to(cuda_device))
    want = ops.linear_fp8(x, w, scale)
    for name in ("_SPLITK_WS", "_SPLITK_OUTGROWN"):
        monkeypatch.setattr(ops, name, {})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.linear_fp8(x, w, scale)
    assert all(torch.equal(a, b) for a, b in zip(ops.linear_fp8(x, w, scale), want))  # before any replay
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
    assert all(torch.equal(a, b) for a, b in zip(ops.linear_fp8(x, w, scale), want))
    assert _lib.device_error() == 0
