"""The serving operators on the host: refusals before anything is launched, the
angle tables against their published formulas, and the 64-bit statements the
GPU tests compare with against torch."""
import ctypes
import math

import numpy as np
import pytest
import torch

import serving_ref as ref
from freemoe_amd import fmx
from freemoe_amd import serving as sv


def buffer():
    buf = np.zeros(4096, np.float32)
    return buf, buf.ctypes.data + (-buf.ctypes.data) % 256


def descriptors(p, **change):
    c = dict(type=fmx.FMX_TYPE_BF16, kv_heads=2, head_dim=64, page_size=16, pages=8, page_stride=2048,
             position_stride=128, head_stride=64, k=p, v=p)
    b = dict(sequences=1, tokens=1, max_new=1, table_stride=4, starts=p, lengths=p, table=p)
    for name, value in change.items():
        (c if name in c else b)[name] = value
    return fmx.PagedCache(*c.values()), fmx.PagedBatch(*b.values())


def attention(p, heads=4, q=None, out=None, out_type=0, q_stride=256, out_stride=256, ws=None, ws_bytes=1 << 40,
              options=(0.125, 0.0, 0, None), **change):
    cache, batch = descriptors(p, **change)
    return fmx.lib().fmx_attention_paged(ctypes.byref(cache), ctypes.byref(batch),
                                         ctypes.byref(fmx.AttentionOptions(*options)), heads, p if q is None else q,
                                         q_stride, out_type, p if out is None else out, out_stride,
                                         p if ws is None else ws, ws_bytes, None)


def rope(p, heads=4, in_type=0, layout=1, dims=64, inv=True, magnitude=1.0, q=None, q_out=None, strides=(512, 512, 512, 256),
         ws_bytes=256, **change):
    cache, batch = descriptors(p, **change)
    r = fmx.Rope(layout, dims, p if inv else None, magnitude, None)
    return fmx.lib().fmx_rope_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(r), heads, in_type,
                                     p if q is None else q, strides[0], p + 4096, strides[1], p + 4096, strides[2],
                                     p + 8192 if q_out is None else q_out, strides[3], p, ws_bytes, None)


SHARED = [
    # what is wrong, status
    (dict(type=fmx.FMX_TYPE_Q8_0), 2), (dict(head_dim=60), 3), (dict(head_dim=264), 3), (dict(head_dim=0), 3),
    (dict(page_size=0), 3), (dict(page_size=65537), 3), (dict(pages=0), 3), (dict(kv_heads=0), 3),
    (dict(page_stride=2044), 3), (dict(position_stride=60), 3), (dict(head_stride=68), 3),
    (dict(page_stride=1 << 40), 3), (dict(table_stride=0), 3), (dict(k=None), 1), (dict(starts=None), 1),
    (dict(lengths=None), 1), (dict(table=None), 1),
]


@pytest.mark.parametrize("change,status", SHARED)
def test_paged_descriptors_refused(change, status):
    buf, p = buffer()
    if "k" in change:
        assert attention(p, **change) == status and attention(p, v=p + 4) == 1
    assert attention(p, **change) == status
    assert rope(p, **change) == status
    cache, batch = descriptors(p, **change)
    assert fmx.lib().fmx_attention_paged_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), 4) == 0


def test_attention_paged_refusals():
    buf, p = buffer()
    assert attention(p, heads=3) == 3 and attention(p, heads=0) == 3 and attention(p, heads=65536) == 3
    assert attention(p, out_type=fmx.FMX_TYPE_F16) == 2
    assert attention(p, q_stride=252) == 3 and attention(p, q_stride=260) == 3
    assert attention(p, out_stride=254) == 3 and attention(p, out_stride=258) == 3
    assert attention(p, q=p + 8) == 1 and attention(p, out=p + 8) == 1 and attention(p, ws=p + 8) == 1
    assert attention(p, ws_bytes=0) == 1
    for options in ((math.nan, 0.0, 0, None), (math.inf, 0.0, 0, None), (1.0, -1.0, 0, None), (1.0, math.nan, 0, None)):
        assert attention(p, options=options) == 1
    cache, batch = descriptors(p)
    lib = fmx.lib()
    one = ctypes.byref(fmx.AttentionOptions(1.0, 0.0, 0, None))
    assert lib.fmx_attention_paged(None, ctypes.byref(batch), one, 4, p, 256, 0, p, 256, p, 1 << 40, None) == 1
    assert lib.fmx_attention_paged(ctypes.byref(cache), None, one, 4, p, 256, 0, p, 256, p, 1 << 40, None) == 1
    assert lib.fmx_attention_paged(ctypes.byref(cache), ctypes.byref(batch), None, 4, p, 256, 0, p, 256, p, 1 << 40, None) == 1
    # nothing to do: no launch, so no GPU is needed
    assert attention(p, tokens=0) == 0 and attention(p, sequences=0) == 0 and attention(p, max_new=0) == 0
    assert attention(p, tokens=1 << 30, max_new=1) == 3  # 2^32 rows of heads


def test_rope_append_refusals():
    buf, p = buffer()
    assert rope(p, layout=2) == 1 and rope(p, magnitude=math.nan) == 1 and rope(p, inv=False) == 1
    assert rope(p, dims=63) == 3 and rope(p, dims=66) == 3 and rope(p, heads=0) == 3
    assert rope(p, in_type=fmx.FMX_TYPE_F16) == 2
    assert rope(p, strides=(252, 512, 512, 256)) == 3 and rope(p, strides=(512, 514, 512, 256)) == 3
    assert rope(p, strides=(512, 512, 64, 256)) == 3 and rope(p, strides=(512, 512, 512, 128)) == 3
    assert rope(p, q=p + 4) == 1 and rope(p, ws_bytes=255) == 1
    assert rope(p, q_out=p, q=p) == 1  # in place needs one type and one stride
    assert rope(p, tokens=0) == 0


def test_sample_refusals():
    buf, p = buffer()
    lib = fmx.lib()
    s = fmx.Sampling(None, None, None, None)

    def sample(logits=p, stride=100, rows=1, vocab=100, settings=ctypes.byref(s), u=p, ids=p, ws=p, ws_bytes=1 << 40):
        return lib.fmx_sample(logits, stride, rows, vocab, settings, u, ids, None, ws, ws_bytes, None)

    assert sample(vocab=0) == 3 and sample(vocab=262145, stride=262145) == 3 and sample(stride=99) == 3
    assert sample(logits=None) == 1 and sample(logits=p + 2) == 1 and sample(u=None) == 1 and sample(ids=None) == 1
    assert sample(settings=None) == 1 and sample(ws=None) == 1 and sample(ws=p + 4) == 1 and sample(ws_bytes=255) == 1
    assert sample(rows=0) == 0
    assert lib.fmx_sample_workspace_bytes(1, 100) >= 256


def test_tensors_that_do_not_fit_are_refused():
    """The tensors' types and shapes, before an address reaches the library."""
    bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    cache = sv.Cache(2, 16, 2, 64, bf16, "cpu")
    batch = sv.Batch(torch.tensor([0, 2], dtype=i32), torch.tensor([5], dtype=i32), torch.zeros(1, 2, dtype=i32), 2, 2)
    rope, ws = sv.Rope(64, device="cpu"), sv.workspace(device="cpu")
    rows = lambda heads, dtype, tokens=2, dim=64: torch.zeros(tokens, heads, dim, dtype=dtype)
    for q, out, more in [(rows(4, f32), rows(4, f32), {}), (rows(4, bf16, 1), rows(4, bf16), {}),
                         (rows(4, bf16, dim=32), rows(4, bf16), {}), (rows(4, bf16), rows(2, bf16), {}),
                         (rows(8, bf16)[:, ::2], rows(4, bf16), {}), (rows(4, bf16, dim=128)[..., ::2], rows(4, bf16), {}),
                         (rows(4, bf16), rows(4, bf16), dict(sinks=torch.zeros(3))),
                         (rows(4, bf16), rows(4, bf16), dict(sinks=torch.zeros(4, dtype=bf16)))]:
        with pytest.raises(ValueError):
            sv.attention(cache, batch, q, out, ws, **more)
    for q, k, v, out, more in [(rows(4, f32), rows(2, bf16), rows(2, f32), rows(4, bf16), {}),
                               (rows(4, f32), rows(2, f32), rows(2, bf16), rows(4, bf16), {}),
                               (rows(4, f32), rows(2, f32), rows(2, f32), rows(4, f32), {}),
                               (rows(4, f32), rows(4, f32), rows(2, f32), rows(4, bf16), {}),
                               (rows(4, f32), rows(2, f32), rows(2, f32, 1), rows(4, bf16), {}),
                               (rows(4, f32), rows(2, f32), rows(2, f32), rows(4, bf16), dict(positions=torch.zeros(2, dtype=torch.int64))),
                               (rows(4, f32), rows(2, f32), rows(2, f32), rows(4, bf16), dict(positions=torch.zeros(1, dtype=i32)))]:
        with pytest.raises(ValueError):
            sv.rope_append(cache, batch, rope, q, k, v, out, ws, **more)
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for logits, uniform, more in [(x.half(), u, {}), (torch.zeros(3, 20)[:, ::2], u, {}), (x, u[:2], {}), (x, u.double(), {}),
                                  (x, torch.zeros(6)[::2], {}), (x, u, dict(top_k=torch.zeros(3))),
                                  (x, u, dict(temperature=torch.zeros(1))), (x, u, dict(ids=torch.zeros(3, dtype=torch.int64)))]:
        with pytest.raises(ValueError):
            sv.sample(logits, uniform, ws, **more)


def test_tensors_that_are_not_on_the_gpu_are_refused():
    """Nothing of what the kernels would read may lie in host memory, or on a GPU
    that is not the current one (here: a device without memory of its own)."""
    i32 = torch.int32
    cache = sv.Cache(2, 16, 2, 64, torch.float32, "cpu")
    batch = sv.Batch(torch.tensor([0, 2], dtype=i32), torch.tensor([5], dtype=i32), torch.zeros(1, 2, dtype=i32), 2, 2)
    rope, ws = sv.Rope(64, device="cpu"), sv.workspace(device="cpu")
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="not the current GPU"):
        sv.attention(cache, batch, q, torch.zeros_like(q), ws)
    with pytest.raises(ValueError, match="not the current GPU"):
        sv.rope_append(cache, batch, rope, q, k, k, torch.zeros_like(q), ws)
    with pytest.raises(ValueError, match="not the current GPU"):
        sv.sample(torch.zeros(1, 4), torch.zeros(1), ws)
    elsewhere = torch.zeros(2, 4, 64, device="meta")
    with pytest.raises(ValueError, match="not meta"):
        sv.attention(cache, batch, q, elsewhere, ws)
    with pytest.raises(ValueError, match="not meta"):
        sv.rope_append(cache, batch, rope, q, k, k, q, ws, positions=torch.zeros(2, dtype=i32, device="meta"))
    with pytest.raises(ValueError, match="not meta"):
        sv.sample(torch.zeros(1, 4), torch.zeros(1, device="meta"), ws)
    with pytest.raises(ValueError, match="alike"):
        sv.Cache.of(cache.k, cache.v.to("meta"))
    with pytest.raises(ValueError, match="one device"):
        sv.Batch(batch.starts, batch.lengths, batch.table.to("meta"), 2, 2)


def frequencies(dims, *scaling):
    inv, magnitude = (ctypes.c_double * (dims // 2))(), ctypes.c_double()
    fmx.call("fmx_rope_frequencies", ctypes.byref(fmx.RopeScaling(*scaling)), dims, inv, ctypes.byref(magnitude))
    return np.array(list(inv)), magnitude.value


def test_rope_frequencies():
    base = 10000.0 ** (-2.0 * np.arange(32) / 64)
    inv, m = frequencies(64, fmx.ROPE_SCALE_NONE, 10000.0, 0.0, 0.0, 0.0, 0.0)
    assert np.allclose(inv, base, rtol=1e-15) and m == 1.0
    inv, m = frequencies(64, fmx.ROPE_SCALE_LINEAR, 10000.0, 4.0, 0.0, 0.0, 0.0)
    assert np.allclose(inv, base / 4, rtol=1e-15) and m == 1.0
    # yarn: pairs that turn over 32 times within the context stay, those under
    # once are divided, and between them every pair lies between the two
    inv, m = frequencies(64, fmx.ROPE_SCALE_YARN, 10000.0, 8.0, 4096.0, 1.0, 32.0)
    turns = 4096.0 * base / (2 * math.pi)
    assert m == pytest.approx(0.1 * math.log(8.0) + 1.0, rel=1e-15)
    low = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    high = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    ramp = np.clip((np.arange(32) - low) / (high - low), 0, 1)
    assert np.allclose(inv, base / 8 * ramp + base * (1 - ramp), rtol=1e-14)
    assert np.allclose(inv[turns > 40], base[turns > 40]) and np.allclose(inv[turns < 0.8], base[turns < 0.8] / 8)
    # bands: by wavelength against context / low and context / high
    inv, m = frequencies(128, fmx.ROPE_SCALE_BANDS, 500000.0, 8.0, 8192.0, 1.0, 4.0)
    f = 500000.0 ** (-2.0 * np.arange(64) / 128)
    wave = 2 * math.pi / f
    blend = (8192.0 / wave - 1.0) / 3.0
    want = np.where(wave < 8192 / 4, f, np.where(wave > 8192, f / 8, (1 - blend) * f / 8 + blend * f))
    assert np.allclose(inv, want, rtol=1e-13) and m == 1.0


@pytest.mark.parametrize("dims,scaling,status", [
    (63, (0, 1e4, 1.0, 0.0, 0.0, 0.0), 3), (0, (0, 1e4, 1.0, 0.0, 0.0, 0.0), 3), (258, (0, 1e4, 1.0, 0.0, 0.0, 0.0), 3),
    (64, (4, 1e4, 1.0, 0.0, 0.0, 0.0), 1), (64, (0, 1.0, 1.0, 0.0, 0.0, 0.0), 1), (64, (0, math.inf, 1.0, 0.0, 0.0, 0.0), 1),
    (64, (1, 1e4, 0.5, 0.0, 0.0, 0.0), 1), (64, (1, 1e4, math.nan, 0.0, 0.0, 0.0), 1),
    (64, (2, 1e4, 2.0, 0.0, 1.0, 32.0), 1), (64, (2, 1e4, 2.0, 4096.0, 32.0, 1.0), 1), (64, (3, 1e4, 2.0, 4096.0, 0.0, 4.0), 1),
])
def test_rope_frequencies_refusals(dims, scaling, status):
    inv, magnitude = (ctypes.c_double * 129)(), ctypes.c_double()
    assert fmx.lib().fmx_rope_frequencies(ctypes.byref(fmx.RopeScaling(*scaling)), dims, inv, ctypes.byref(magnitude)) == status
    assert fmx.lib().fmx_rope_frequencies(None, 64, inv, ctypes.byref(magnitude)) == 1


def test_status_word_of_a_bad_page():
    assert fmx.lib().fmx_moe_status_of(4) == 1 and fmx.lib().fmx_moe_status_of(5) == 1


def test_the_attention_statement_against_softmax():
    P = ref.Paged([3, 2], [9, 2], 2, 8, 4, torch.float32, 1)
    q = torch.randn(P.tokens, 4, 8, generator=P.g)
    for i, (rows, out, _, _) in enumerate(ref.attention(P, q, 0.3)):
        k = P.rows(i, 0).double().repeat_interleave(2, dim=1).transpose(0, 1)
        v = P.rows(i, 1).double().repeat_interleave(2, dim=1).transpose(0, 1)
        n, length = P.counts[i], P.lengths[i]
        mask = torch.ones(n, length, dtype=torch.bool).tril(length - n)
        s = (q[rows].double().transpose(0, 1) @ k.transpose(1, 2) * 0.3).masked_fill(~mask, -math.inf)
        assert torch.allclose((torch.softmax(s, -1) @ v).transpose(0, 1), out, rtol=1e-12)


def test_the_rope_statement_turns_by_its_angle():
    x = torch.randn(5, 2, 16)
    inv = torch.tensor([1.0, 0.5, 0.1], dtype=torch.float64)
    pos = torch.tensor([0, 1, 2, 100, 7])
    for half in (False, True):
        out, _ = ref.rope(x, pos, inv, 2.0, 6, half)
        a, b = (slice(0, 3), slice(3, 6)) if half else (slice(0, 6, 2), slice(1, 6, 2))
        z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.polar(torch.full((5, 3), 2.0, dtype=torch.float64), pos[:, None] * inv)[:, None]
        assert torch.allclose(out[..., a], z.real) and torch.allclose(out[..., b], z.imag)
        assert torch.equal(out[..., 6:], x[..., 6:].double())
