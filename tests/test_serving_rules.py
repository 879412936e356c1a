"""What the serving module and calls promise beside their values, on the host."""
import contextlib
import ctypes
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


@pytest.fixture
def buffer():
    """An aligned host address that no refused call reads."""
    data = torch.zeros(4096)
    return data, data.data_ptr() + (-data.data_ptr()) % 256


def attention(p, heads=4, tokens=0, max_new=1, options=(0.125, 0.0, 0, None), out_stride=256, **batch):
    """fmx_attention_paged on descriptors without work unless `tokens` says so."""
    cache = fmx.PagedCache(fmx.FMX_TYPE_BF16, 2, 64, 16, 8, 2048, 128, 64, p, p)
    b = dict(sequences=1, tokens=tokens, max_new=max_new, table_stride=4, starts=p, lengths=p, table=p)
    b.update(batch)
    return fmx.lib().fmx_attention_paged(ctypes.byref(cache), ctypes.byref(fmx.PagedBatch(*b.values())),
                                         ctypes.byref(fmx.AttentionOptions(*options)), heads, p, 256, 0, p, out_stride, p,
                                         1 << 62, None)


def test_softcaps_that_a_float_does_not_hold_are_refused(buffer):
    """Below a float's normal values, or with a scale over it that passes them, the
    kernels would leave the cap out or turn scores of 0 into NaN."""
    _, p = buffer
    for scale, cap in ((0.125, 1e-46), (0.125, 5e-324), (0.0, 1e-50), (0.125, 1e-39), (-1e25, 1e-20), (1e30, 1e-10), (2.0 ** 99, 2.0 ** -28)):
        assert attention(p, options=(scale, cap, 0, None)) == 1, (scale, cap)
    for scale, cap in ((0.125, 1e-30), (0.0, 2.0 ** -126), (-1e20, 1e-10), (0.125, 50.0), (1e-300, 2.0 ** 99), (2.0 ** 99, 1.0), (1.0, 0.0)):
        assert attention(p, options=(scale, cap, 0, None)) == 0, (scale, cap)  # (nothing to do: no launch)


def test_calls_larger_than_a_launch_are_refused(buffer):
    """A launch takes fewer than 2^32 threads in a dimension: refused by size before
    anything is launched, as any other shape."""
    _, p = buffer
    lib = fmx.lib()
    cache = fmx.PagedCache(fmx.FMX_TYPE_BF16, 2, 64, 16, 8, 2048, 128, 64, p, p)
    for tokens in (1 << 24, 1 << 30, (1 << 31) - 1):
        batch = fmx.PagedBatch(1, tokens, tokens, 4, p, p, p)
        turn = fmx.Rope(1, 64, p, 1.0, None)
        assert lib.fmx_rope_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(turn), 4, 0, p, 512, p, 512, p,
                                   512, p, 256, p, 256, None) == 3
    settings = fmx.Sampling(None, None, None, None)
    for rows in (1 << 23, 1 << 24, (1 << 31) - 1, (1 << 32) - 1):
        assert lib.fmx_sample(p, 100, rows, 100, ctypes.byref(settings), p, p, None, p, 1 << 62, None) == 3
    # single tokens of as many sequences: a tile each, and kv heads times that
    assert attention(p, tokens=1 << 23, sequences=1 << 23) == 3
    # one prompt: 128 rows a tile, 2 kv heads
    assert attention(p, tokens=(1 << 29) - 1, max_new=1 << 29) == 3


def test_the_status_of_what_is_no_workspace_is_refused(monkeypatch):
    """The word is cleared by a kernel: it has to be the current GPU's memory."""
    monkeypatch.setattr(fmx, "lib", lambda: pytest.fail("an address of the host reached the library"))
    monkeypatch.setattr(fmx, "stream_handle", lambda stream=None: 0)
    with pytest.raises(ValueError, match="not the current GPU"):
        sv.status(sv.workspace(device="cpu"))
    with pytest.raises(ValueError, match="256 entries"):
        sv.status(torch.zeros(2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="uint8"):
        sv.status(torch.zeros(256))
