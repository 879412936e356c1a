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


def test_a_stream_of_another_device_is_refused():
    i32 = torch.int32
    cache = sv.Cache(2, 16, 2, 64, torch.float32, "cpu")
    batch = sv.Batch(torch.tensor([0, 2], dtype=i32), torch.tensor([5], dtype=i32), torch.zeros(1, 2, dtype=i32), 2, 2)
    rope, ws = sv.Rope(64, device="cpu"), sv.workspace(device="cpu")
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    other = types.SimpleNamespace(cuda_stream=7, device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="a stream of cuda:1"):
        sv.attention(cache, batch, q, torch.zeros_like(q), ws, stream=other)
    with pytest.raises(ValueError, match="a stream of cuda:1"):
        sv.rope_append(cache, batch, rope, q, k, k, torch.zeros_like(q), ws, stream=other)
    for given in (ws, None):
        with pytest.raises(ValueError, match="a stream of cuda:1"):
            sv.sample(torch.zeros(1, 4), torch.zeros(1), given, stream=other)
