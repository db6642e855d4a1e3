"""device_error() after a device-side timeout: what the hooks issue has finished when it returns. No GPU: a fake library."""
import torch

from whisper_blaze_b200 import _lib


class Library:
    def __init__(self, word):
        self.word = word

    def wbk_device_error(self, out):
        out._obj.value = self.word
        return 0


def test_the_hooks_work_is_waited_for(monkeypatch):
    log = []
    monkeypatch.setattr(_lib, "_TIMEOUT_HOOKS", [lambda dev: log.append(("hook", dev))])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda dev=None: log.append(("wait", dev)))
    monkeypatch.setattr(_lib, "lib", lambda: Library(_lib.WBK_ERR_DEVICE_TIMEOUT | 41 << 8))
    assert _lib.device_error() == _lib.WBK_ERR_DEVICE_TIMEOUT | 41 << 8
    assert log == [("hook", 3), ("wait", 3)]
    log.clear()
    monkeypatch.setattr(_lib, "lib", lambda: Library(0))
    assert _lib.device_error() == 0 and not log
