"""The serving operators driven through libfmx on torch tensors: a paged cache
in HBM, rotary positions with the cache write, attention over the pages, and
sampling.

torch provides the device memory and the stream; every computation is a
libfmx call. Sequences, their lengths and their pages are the caller's: a
Batch holds the device arrays that name them, and a captured graph follows
what those hold at each replay.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import fmx

TYPE_IDS = {torch.float32: fmx.FMX_TYPE_F32, torch.float16: fmx.FMX_TYPE_F16, torch.bfloat16: fmx.FMX_TYPE_BF16}


class Cache:
    """One layer's keys and values: `pages` pages of `page_size` positions."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        self.k = torch.zeros(pages, page_size, kv_heads, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.describe()

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor) -> "Cache":
        """On existing pools, [page, place, kv head, element] with any strides the library takes."""
        if (k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device
                or k.dim() != 4 or k.stride(3) != 1):
            raise ValueError("k and v: alike, [page, place, kv head, element], elements next to each other")
        self = cls.__new__(cls)
        self.k, self.v = k, v
        self.describe()
        return self

    def describe(self):
        pages, page_size, kv_heads, head_dim = self.k.shape
        # (torch gives dimensions of one entry any stride)
        strides = [s if n > 1 else self.k.numel() for s, n in zip(self.k.stride(), self.k.shape)]
        strides = [-(-max(s, head_dim) // 8) * 8 if n == 1 else s for s, n in zip(strides, self.k.shape)]
        self.desc = fmx.PagedCache(TYPE_IDS[self.k.dtype], kv_heads, head_dim, page_size, pages, strides[0], strides[1],
                                   strides[2], self.k.data_ptr(), self.v.data_ptr())


class Batch:
    """The new tokens of a step: starts [sequences + 1], lengths [sequences] and
    table [sequences, pages of the longest], int32 on the device."""

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, tokens: int, max_new: int):
        for t in (starts, lengths, table):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != starts.device:
                raise ValueError("starts, lengths and table: contiguous int32 on one device")
        if starts.numel() != lengths.numel() + 1 or table.shape[0] != lengths.numel():
            raise ValueError("starts: one more than lengths; table: a row per sequence")
        self.starts, self.lengths, self.table, self.tokens = starts, lengths, table, tokens
        self.device = starts.device
        self.desc = fmx.PagedBatch(lengths.numel(), tokens, max_new, table.shape[1], starts.data_ptr(),
                                   lengths.data_ptr(), table.data_ptr())


class Rope:
    """The angles of a model: made once on the host, kept on the device."""

    def __init__(self, dims: int, base: float = 10000.0, layout: int = fmx.ROPE_HALF, kind: int = fmx.ROPE_SCALE_NONE,
                 factor: float = 1.0, context: float = 0.0, low: float = 1.0, high: float = 32.0, device="cuda"):
        scaling = fmx.RopeScaling(kind, base, factor, context, low, high)
        inv, magnitude = (ctypes.c_double * (dims // 2))(), ctypes.c_double()
        fmx.call("fmx_rope_frequencies", ctypes.byref(scaling), dims, inv, ctypes.byref(magnitude))
        self.inv_freq = torch.tensor(list(inv), dtype=torch.float64, device=device)
        self.layout, self.dims, self.magnitude = layout, dims, magnitude.value

    def desc(self, positions=None):  # positions: a device address
        return fmx.Rope(self.layout, self.dims, self.inv_freq.data_ptr(), self.magnitude, positions)


def _rows(t: torch.Tensor, device, tokens: int, heads: int, head_dim: int, dtype=None) -> int:
    """Row stride of [tokens, heads, head_dim] (the heads of a row next to each other)."""
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if n < tokens or h != heads or d != head_dim or s2 != 1 or (h > 1 and s1 != d):
        raise ValueError("rows: [tokens, heads, head_dim], a row's heads next to each other")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"rows of {dtype}, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"rows on {device}, not {t.device}")
    return s0 if n > 1 else h * d  # (one row's stride is never used, and torch may give it any)


def _entries(t: torch.Tensor | None, device, count: int, dtype):
    """A device array of `count` entries, or NULL."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() < count or not t.is_contiguous():
        raise ValueError(f"an array of {count} entries of {dtype}, next to each other")
    if t.device != device:
        raise ValueError(f"an array on {device}, not {t.device}")
    return t.data_ptr()


def _same_gpu(device, stream):
    """A stream of another GPU would run the kernels there. (What only has a handle is taken, as by stream_handle.)"""
    if getattr(stream, "device", device) != device:
        raise ValueError(f"a stream of {stream.device} for tensors on {device}")


def _stream(device, stream, *others):
    """The stream's handle; its GPU, which is the current one, must hold the tensors."""
    _same_gpu(device, stream)
    for other in others:
        if other != device:
            raise ValueError(f"tensors on {device} and on {other}")
    if device.type != "cuda" or device.index != torch.cuda.current_device():
        raise ValueError(f"tensors on {device}, which is not the current GPU")
    return fmx.stream_handle(stream)


def workspace(bytes_: int = 256, device="cuda") -> torch.Tensor:
    """Zeroed on the current stream, for which a call on another stream has to wait."""
    return torch.zeros(bytes_, dtype=torch.uint8, device=device)


def status(ws: torch.Tensor, stream=None) -> int:
    """The error word's status; clears it. Waits for the stream."""
    word, handle = _entries(ws, ws.device, 256, torch.uint8), _stream(ws.device, stream)
    return fmx.lib().fmx_moe_status(word, handle)


def rope_append(cache: Cache, batch: Batch, rope: Rope, q, k, v, q_out, ws, positions=None, stream=None):
    n, heads, kv_heads, d, dtype = batch.tokens, q.shape[1], cache.desc.kv_heads, cache.desc.head_dim, q.dtype
    dev = cache.k.device
    fmx.call("fmx_rope_append", ctypes.byref(cache.desc), ctypes.byref(batch.desc),
             ctypes.byref(rope.desc(_entries(positions, dev, n, torch.int32))), heads, TYPE_IDS[dtype], q.data_ptr(),
             _rows(q, dev, n, heads, d), k.data_ptr(), _rows(k, dev, n, kv_heads, d, dtype), v.data_ptr(),
             _rows(v, dev, n, kv_heads, d, dtype), q_out.data_ptr(), _rows(q_out, dev, n, heads, d, cache.k.dtype),
             _entries(ws, dev, 0, torch.uint8), ws.numel(), _stream(dev, stream, batch.device, rope.inv_freq.device))
    return q_out


def attention_workspace(cache: Cache, batch: Batch, heads: int) -> torch.Tensor:
    need = fmx.lib().fmx_attention_paged_workspace_bytes(ctypes.byref(cache.desc), ctypes.byref(batch.desc), heads)
    if need == 0:
        raise fmx.FmxError(1, "fmx_attention_paged_workspace_bytes")
    return workspace(need, cache.k.device)


def attention(cache: Cache, batch: Batch, q, out, ws, scale=None, softcap=0.0, window=0, sinks=None, stream=None):
    n, heads, d, dev = batch.tokens, q.shape[1], cache.desc.head_dim, cache.k.device
    options = fmx.AttentionOptions(1.0 / math.sqrt(d) if scale is None else scale, softcap, window,
                                   _entries(sinks, dev, heads, torch.float32))
    fmx.call("fmx_attention_paged", ctypes.byref(cache.desc), ctypes.byref(batch.desc), ctypes.byref(options), heads,
             q.data_ptr(), _rows(q, dev, n, heads, d, cache.k.dtype), TYPE_IDS[out.dtype], out.data_ptr(),
             _rows(out, dev, n, heads, d), _entries(ws, dev, 0, torch.uint8), ws.numel(),
             _stream(dev, stream, batch.device))
    return out


class Sampled(tuple):
    """(ids, probs), with the workspace whose error word reports the rows without a distribution."""

    def __new__(cls, ids, probs, ws):
        self = super().__new__(cls, (ids, probs))
        self.ids, self.probs, self.ws = ids, probs, ws
        return self


def sample(logits, uniform, ws=None, temperature=None, top_k=None, top_p=None, min_p=None, ids=None, probs=None,
           stream=None):
    """Token ids (int32) and their probabilities, one per row of logits. A row
    without a distribution has id -1 and probability 0, and is reported by
    status(ws), of the result's own `ws` where none is given. What is not given is
    made on the call's stream, and belongs to it as any tensor of torch does."""
    rows, vocab = logits.shape
    if logits.dtype != torch.float32 or (vocab > 1 and logits.stride(1) != 1):
        raise ValueError("logits: float32 rows")
    _same_gpu(logits.device, stream)
    # (another stream's blocks may still be written there, and a workspace that ends
    # with this call may be handed out again while the kernel runs)
    with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
        ids = torch.empty(rows, dtype=torch.int32, device=logits.device) if ids is None else ids
        probs = torch.empty(rows, dtype=torch.float32, device=logits.device) if probs is None else probs
        ws = workspace(fmx.lib().fmx_sample_workspace_bytes(rows, vocab), logits.device) if ws is None else ws
    dev, f32, i32 = logits.device, torch.float32, torch.int32
    settings = fmx.Sampling(_entries(temperature, dev, rows, f32), _entries(top_k, dev, rows, i32),
                            _entries(top_p, dev, rows, f32), _entries(min_p, dev, rows, f32))
    fmx.call("fmx_sample", logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab,
             ctypes.byref(settings), _entries(uniform, dev, rows, f32), _entries(ids, dev, rows, i32),
             _entries(probs, dev, rows, f32), _entries(ws, dev, 0, torch.uint8), ws.numel(), _stream(dev, stream))
    return Sampled(ids, probs, ws)
