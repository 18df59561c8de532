"""CPU: every stream of a step is asked for at the normal priority, whatever the environment holds."""
import contextlib
import types

import torch

from helpers import pkg


def test_the_side_stream_has_normal_priority(monkeypatch):
    E = pkg("engine")
    asked = []
    fake = types.SimpleNamespace(srx_stream_create=lambda priority, out: asked.append(priority) or 0)
    monkeypatch.setattr(E.L, "lib", lambda: fake)
    monkeypatch.setattr(E, "_SIDE_STREAMS", {})
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda pointer, device: object())
    monkeypatch.setenv("SRX_SIDE_STREAM_PRIORITY", "1")
    first = E.side_stream(torch.device("cuda", 0))
    assert asked == [0] and E.side_stream(torch.device("cuda", 0)) is first
