"""The extension module with the short way to the decoder-step calls: where it cannot be used, the calls do without."""
import importlib.util
import os

import pytest
import torch

from whisper_blaze_b200 import _lib, ops


def _build_py():
    """csrc/build.py as a module of its own."""
    path = os.path.join(os.path.dirname(os.path.dirname(_lib.LIB_PATH)), "csrc", "build.py")
    spec = importlib.util.spec_from_file_location("wbk_build", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


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


def test_a_module_for_another_torch_is_done_without_and_built_anew(tmp_path, monkeypatch):
    build = _build_py()
    src = os.path.join(build.HERE, "wbk_calls.cpp")
    assert _lib.calls().built_for == build.calls_for()
    other = tmp_path / "for"
    monkeypatch.setattr(build, "CALLS_FOR", str(other))
    monkeypatch.setattr(build, "_stale", lambda *_: False)  # no source is newer
    assert build._calls_stale(src)
    for text, stale in ((build.calls_for(), False), (build.calls_for().replace(torch.__version__, "2.0.0"), True)):
        other.write_text(text)
        assert build._calls_stale(src) is stale
    monkeypatch.setattr(torch, "__version__", "2.0.0")
    assert _lib.calls() is None


def test_the_library_is_built_where_the_module_is_not(tmp_path, monkeypatch, capsys):
    """No g++: everything but the module is linked, and the reason is printed."""
    build = _build_py()
    linked = []

    def run(cmd, **_):
        if cmd[0].endswith("g++"):
            raise FileNotFoundError("g++")
        linked.append(cmd)
        return type("Done", (), {"returncode": 0, "stdout": "", "stderr": ""})

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "_calls_stale", lambda src: True)
    for name, file in (("BUILD", ""), ("LIB", "libwbk.so"), ("CALLS", "_wbk_calls.so"), ("CALLS_FOR", "for")):
        monkeypatch.setattr(build, name, str(tmp_path / file))
    (tmp_path / "_wbk_calls.so").write_bytes(b"of another torch")
    assert build.build() == build.LIB
    assert "-shared" in linked[-1] and build.LIB in linked[-1]
    assert not (tmp_path / "_wbk_calls.so").exists()  # a stale one does not stay
    assert "_wbk_calls.so is not built" in capsys.readouterr().err
