"""What the serving module and calls promise beside their values, on the host."""
import contextlib
import types

import pytest
import torch

from freemoe_amd import fmx
from freemoe_amd import serving as sv


def test_sample_makes_its_tensors_on_the_calls_stream(monkeypatch):
    """Ids, probabilities and the workspace that a call makes come from the memory of
    the stream it runs on, and the workspace lives as long as its result."""
    on, made, calls = [None], [], []

    @contextlib.contextmanager
    def enter(stream):
        on.append(stream)
        yield
        on.pop()

    def recorded(make):
        def wrapped(*a, **kw):
            made.append(on[-1])
            return make(*a, **kw)
        return wrapped

    monkeypatch.setattr(torch.cuda, "stream", enter)
    monkeypatch.setattr(torch, "empty", recorded(torch.empty))
    monkeypatch.setattr(torch, "zeros", recorded(torch.zeros))
    monkeypatch.setattr(sv, "_stream", lambda device, stream, *others: 0)
    monkeypatch.setattr(fmx, "call", lambda name, *a: calls.append((name, on[-1])))
    x, u = torch.randn(3, 10), torch.rand(3)
    for stream in (None, types.SimpleNamespace(cuda_stream=7)):
        made.clear()
        got = sv.sample(x, u, stream=stream)
        assert made == [stream] * 3 and calls.pop()[0] == "fmx_sample"
        ids, probs = got
        assert ids is got.ids and probs is got.probs and got.ws.dtype == torch.uint8 and got.ws.numel() >= 256
    ws = torch.zeros(256, dtype=torch.uint8)
    assert sv.sample(x, u, ws).ws is ws
