"""The extension module with the short way to the decoder-step calls: where it cannot be used, the calls do without."""
import os

import pytest
import torch

from whisper_blaze_b200 import _lib, ops


def test_the_built_module_loads():
    assert _lib.calls() is not None


def test_a_module_that_does_not_load_is_done_without(tmp_path, monkeypatch):
    """An undefined symbol (the module of another torch) and a file that is no library are ImportErrors of the loader."""
    broken = tmp_path / "_wbk_calls.so"
    broken.write_bytes(b"\x7fELF no library")
    monkeypatch.setattr(_lib, "CALLS_PATH", str(broken))
    assert _lib.calls() is None
    monkeypatch.setattr(ops, "_SHORT", [])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):  # ops.py's own checks
        ops.sample(torch.zeros(1, 5), torch.ones(1, 5))
    monkeypatch.setattr(_lib, "CALLS_PATH", os.path.join(str(tmp_path), "nothing.so"))
    assert _lib.calls() is None
