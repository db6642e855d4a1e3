"""Decoders of one device take turns on the GPU: the order of what they issue, with recorded streams and events in
place of torch's. No GPU."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from whisper_blaze_b200 import decoding


class Stream:
    def __init__(self, name, log):
        self.name, self.log = name, log

    def wait_event(self, event):
        self.log.append((self.name, "waits", event.behind))


@pytest.fixture
def gpu(monkeypatch):
    """A device whose streams write to `log`; gpu.now is the current stream."""
    log = []
    state = SimpleNamespace(log=log, capturing=False, now=None, a=Stream("a", log), b=Stream("b", log))

    class Event:
        behind = None

        def record(self, stream):
            self.behind = f"{stream.name}{sum(1 for e in log if e[:2] == (stream.name, 'runs'))}"

    monkeypatch.setattr(decoding, "_LAST", {}, raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: state.now)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    return state


class Decoder(decoding.Kv8Decoder):
    """Its logits() is one entry of the log; the rest is Kv8Decoder's."""

    def __init__(self, gpu):
        self.gpu, self.device = gpu, torch.device("cuda", 0)

    def work(self):
        self.gpu.log.append((self.gpu.now.name, "runs"))


def _call(decoder, stream):
    decoder.gpu.now = stream
    with decoding._turn(decoder.device):
        decoder.work()


def test_a_call_waits_for_those_on_other_streams(gpu):
    one, two = Decoder(gpu), Decoder(gpu)
    for decoder, stream in ((one, gpu.a), (two, gpu.b), (two, gpu.b), (one, gpu.a)):
        _call(decoder, stream)
    assert gpu.log == [("a", "runs"), ("b", "waits", "a1"), ("b", "runs"), ("b", "runs"), ("a", "waits", "b2"), ("a", "runs")]


def test_every_public_call_takes_its_turn(gpu):
    """A call that fails before it issues anything still has waited, and leaves an event behind it."""
    _call(Decoder(gpu), gpu.a)
    for call in (lambda d: d.start(None), lambda d: d.logits(None), lambda d: d.step(None), lambda d: d.generate(None, None, 1)):
        gpu.log.clear()
        _call(Decoder(gpu), gpu.a)
        gpu.now = gpu.b
        with pytest.raises(AttributeError):
            call(Decoder(gpu))
        assert gpu.log[-1] == ("b", "waits", "a1") and decoding._LAST[0][0] is gpu.b


def test_inside_a_capture_nothing_is_waited_for(gpu):
    _call(Decoder(gpu), gpu.a)
    gpu.capturing = True
    _call(Decoder(gpu), gpu.b)
    assert gpu.log == [("a", "runs"), ("b", "runs")] and decoding._LAST[0][0] is gpu.a
