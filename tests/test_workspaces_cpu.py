"""The shared workspaces' bookkeeping, on the CPU: ops._zeros makes them here, no kernel runs."""
import gc
import weakref

import pytest
import torch

from whisper_blaze_b200 import ops

DEV = torch.device("cuda", 0)


@pytest.fixture
def made(monkeypatch):
    """Weak references to the tensors that ops made, in order."""
    refs = []

    def zeros(nbytes, device):
        t = torch.zeros(nbytes, dtype=torch.uint8)
        refs.append(weakref.ref(t))
        return t

    monkeypatch.setattr(ops, "_zeros", zeros)
    for name in ("_SPLITK_WS", "_SPLITK_OUTGROWN"):
        monkeypatch.setattr(ops, name, {}, raising=False)
    return refs


def test_an_outgrown_workspace_is_kept(made):
    """A captured graph holds the address of the workspace that its linears had; freed, its memory would be another
    tensor's when the graph is replayed."""
    sizes = [256, 256, 4096, 1 << 20, 512]
    for n in sizes:
        assert ops.splitk_workspace(DEV, n).numel() >= n
    gc.collect()
    assert len(made) == 3 and all(r() is not None for r in made)
    assert ops.splitk_workspace(DEV, 1 << 20) is made[-1]()
    assert sum(r().numel() for r in made) <= 2 * made[-1]().numel()  # what is kept is bounded by the last


def test_a_timeout_zeroes_every_workspace_kept(made):
    for n in (256, 1024, 65536):
        ops.splitk_workspace(DEV, n)
    for r in made:
        r().fill_(0x5A)
    ops._zero_shared_workspaces(0)
    assert len(made) == 3 and all(int(r().count_nonzero()) == 0 for r in made)
