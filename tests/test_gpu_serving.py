"""fmx_rope_append, fmx_attention_paged and fmx_sample against plain statements
in 64 bits, on an MI355X.

Tolerances. A rotated element is a float computation on cosines and sines each
rounded to float: four roundings of 2^-24 of its pair's |x| + |y|, then half a
step of the cache's type. An attention output's error is its weights' relative
error times sum_j p_j |v_j|: twice the score's own (numerator and denominator),
a dot of D products summed in f32 with at most D + 8 roundings of 2^-24 of
sum |q k|, plus 2^-24 for each of the n sums and a few for exponentials and
scaling; where the result has 16 bits, half a step of it, and half a step of
each weight. Every bound is a worst case."""
import math

import numpy as np
import pytest
import torch

import serving_ref as ref
from freemoe_amd import fmx
from freemoe_amd import serving as sv

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def to(gpu, t):
    return None if t is None else t.to(gpu)


# -------------------------------------------------------------------- rope --

ROPE = {
    # name: (heads, kv heads, head_dim, dims, layout, in, cache, page, counts, lengths, by_head)
    "one_token": (4, 2, 64, 64, "half", F32, BF16, 16, [1], [1], False),
    "far": (2, 1, 128, 128, "interleaved", F32, F32, 16, [3], [30001], False),
    "partial_half": (3, 1, 80, 32, "half", F32, F16, 5, [7, 1, 0, 12], [9, 100, 3, 12], False),
    "partial_pairs": (5, 5, 96, 48, "interleaved", BF16, BF16, 24, [30, 2], [30, 77], True),
    "odd_dims": (2, 2, 40, 20, "half", F32, BF16, 1, [4, 4], [6, 5], False),
    "odd_dims_pairs": (2, 2, 24, 6, "interleaved", F16, F16, 3, [5], [11], True),
    "no_dims": (2, 1, 16, 0, "half", F32, F32, 4, [5], [5], False),
    "many_sequences": (2, 1, 64, 64, "half", F32, BF16, 8, [1 + i % 3 for i in range(150)], [1 + i % 3 + i % 40 for i in range(150)], False),
    "widest": (2, 2, 256, 256, "half", F32, BF16, 16, [9], [40], False),
    "long": (2, 1, 64, 32, "half", F32, F16, 64, [700], [700], False),
}


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("name", list(ROPE))
def test_rope_append(gpu, name, fused):
    H, G, D, R, layout, tin, tc, ps, counts, lengths, by_head = ROPE[name]
    P = ref.Paged(counts, lengths, G, D, ps, tc, 11, by_head=by_head, pad=8 if fused else 0)
    x = torch.randn(P.tokens, H + 2 * G, D, generator=P.g).to(tin)
    rope = sv.Rope(R, layout=fmx.ROPE_HALF if layout == "half" else fmx.ROPE_INTERLEAVED, kind=fmx.ROPE_SCALE_YARN,
                   factor=4.0, context=2048.0, device=gpu) if R else None
    if rope is None:
        rope = sv.Rope(2, device=gpu)
        rope.dims = 0
    before = [pool.clone() for pool, _ in P.pools]
    cache, batch = P.on(gpu)
    xd = x.to(gpu)
    q, k, v = (xd[:, :H], xd[:, H:H + G], xd[:, H + G:]) if fused else (xd[:, :H].contiguous(), xd[:, H:H + G].contiguous(), xd[:, H + G:].contiguous())
    out = torch.full((P.tokens, H, D), 7.0, dtype=tc, device=gpu)
    ws = sv.workspace(device=gpu)
    sv.rope_append(cache, batch, rope, q, k, v, out, ws)
    assert sv.status(ws) == 0
    got, pools = out.cpu(), [cache.k.cpu(), cache.v.cpu()]
    want_pools = [b[..., :D].transpose(1, 2).clone() if by_head else b[..., :D].clone() for b in before]
    half, inv = layout == "half", rope.inv_freq.cpu()[:R // 2]
    for i, n in enumerate(counts):
        rows = slice(P.starts[i], P.starts[i] + n)
        pos = torch.arange(lengths[i] - n, lengths[i])
        want, size = ref.rope(x[rows, :H + G], pos, inv, rope.magnitude, R, half)
        tol = 4 * U * size + ref.half_step(tc, want.abs() + 4 * U * size)
        assert ((got[rows].double() - want[:, :H]).abs() <= tol[:, :H]).all(), f"q of sequence {i}"
        page = P.table[i].long()[pos // ps]
        kk = pools[0][page, pos % ps].double()
        assert ((kk - want[:, H:]).abs() <= tol[:, H:]).all(), f"k of sequence {i}"
        assert torch.equal(pools[1][page, pos % ps], x[rows, H + G:].to(tc)), f"v of sequence {i}"
        want_pools[0][page, pos % ps] = pools[0][page, pos % ps]
        want_pools[1][page, pos % ps] = pools[1][page, pos % ps]
    assert (got[P.starts[-1]:] == 7.0).all()  # rows behind the last sequence
    for g, w in zip(pools, want_pools):  # everything else in the pools stays
        assert torch.equal(torch.nan_to_num(g, 123.0), torch.nan_to_num(w, 123.0))


def test_rope_append_at_given_positions_and_in_place(gpu):
    H, G, D, T = 4, 2, 64, 9
    P = ref.Paged([5, 4], [5, 20], G, D, 4, F32, 3)
    x = torch.randn(P.tokens, H + 2 * G, D, generator=P.g)
    positions = torch.tensor([0, 1000000, 3, 70000, 2 ** 30, 5, 5, 5, -6, 0, 0], dtype=torch.int32)
    rope = sv.Rope(D, layout=fmx.ROPE_INTERLEAVED, device=gpu)
    cache, batch = P.on(gpu)
    xd = x.to(gpu)
    ws = sv.workspace(device=gpu)
    sv.rope_append(cache, batch, rope, xd[:, :H], xd[:, H:H + G], xd[:, H + G:], xd[:, :H], ws, positions=positions.to(gpu))
    assert sv.status(ws) == 0
    want, size = ref.rope(x[:T, :H], positions[:T], rope.inv_freq.cpu(), 1.0, D, False)
    got = xd.cpu()
    # an angle of 2^30 radians is exact to 2^-23 as a double product: a few units of 2^-24 more
    assert ((got[:T, :H].double() - want).abs() <= (8 * U) * size + U * want.abs()).all()
    assert torch.equal(got[:, H:], x[:, H:]) and torch.equal(got[T:], x[T:])


def test_rope_append_reports_what_it_does_not_follow(gpu):
    """Pages outside the pool, more new tokens than positions or than max_new and
    starts that fall: reported, those tokens skipped, the others as ever."""
    H = G = 1
    D = 16

    def run(change):
        P = ref.Paged([2, 2, 2], [2, 6, 2], G, D, 2, F32, 5)
        change(P)
        cache, batch = P.on(gpu)
        x = torch.randn(P.tokens, 3, D, generator=P.g).to(gpu)
        out = torch.full((P.tokens, H, D), 7.0, device=gpu)
        ws = sv.workspace(device=gpu)
        rope = sv.Rope(D, device=gpu)
        sv.rope_append(cache, batch, rope, x[:, :1], x[:, 1:2], x[:, 2:], out, ws)
        st = sv.status(ws)
        assert sv.status(ws) == 0  # read and cleared
        return st, [bool((out[i] != 7.0).any()) for i in range(P.tokens)]

    def page(P):
        P.table[1, 2] = 10 ** 6

    def short(P):
        P.lengths = [2, 1, 2]

    def falling(P):
        P.starts = [0, 2, 1, 4]
        P.max_new = 2

    def long(P):
        P.lengths = [2, 10 ** 6, 2]

    def many(P):
        P.max_new = 1

    assert run(lambda P: None) == (0, [True] * 6 + [False] * 2)
    assert run(page) == (1, [True, True, False, False, True, True, False, False])
    assert run(short) == (1, [True, True, False, True, True, True, False, False])
    assert run(long) == (1, [True, True, False, False, True, True, False, False])
    assert run(falling)[0] == 1
    assert run(many) == (1, [False] * 8)


# --------------------------------------------------------------- attention --

ATTENTION = {
    # name: (heads, kv heads, head_dim, cache, out, page, counts, lengths, options)
    "one": (1, 1, 8, F32, F32, 16, [1], [1], {}),
    "decode": (8, 2, 64, BF16, F32, 16, [1, 1, 1, 1], [1, 37, 200, 513], {}),
    "decode_wide_f32": (4, 4, 256, F32, F32, 7, [1, 1], [300, 33], {}),
    "decode_mqa": (20, 1, 128, F16, F16, 16, [1, 1, 1], [999, 64, 65], {}),
    "decode_padded_dim": (6, 3, 80, F16, F32, 24, [1, 1], [129, 257], {}),
    "few_tokens": (4, 2, 96, BF16, BF16, 5, [3, 1, 0, 4], [40, 1, 9, 4], {}),
    "prompt": (4, 2, 64, BF16, BF16, 16, [100], [100], {}),
    "prompt_f32": (2, 1, 128, F32, F32, 16, [70, 5], [70, 133], {}),
    "prompt_f16_f32_out": (2, 2, 128, F16, F32, 32, [65], [90], {}),
    "prompt_wide": (2, 1, 256, BF16, F32, 16, [40], [75], {}),
    "prompt_wide_f16": (2, 1, 192, F16, F16, 16, [33], [75], {}),
    "prompt_narrow": (4, 4, 16, BF16, BF16, 3, [50, 20], [50, 61], {}),
    "prompt_f32_odd": (3, 3, 40, F32, F32, 1, [37], [50], {}),
    "chunk_of_long": (8, 1, 64, BF16, BF16, 64, [33], [1500], {}),
    "window": (4, 2, 64, BF16, F32, 16, [60, 1, 1], [300, 300, 4], dict(window=50)),
    "window_one": (2, 1, 64, F32, F32, 16, [20], [40], dict(window=1)),
    "window_wider_than_all": (2, 1, 32, F16, F16, 16, [20], [40], dict(window=10 ** 9)),
    "window_prompt": (4, 2, 128, BF16, BF16, 16, [200], [200], dict(window=33)),
    "window_f32": (2, 2, 96, F32, F32, 24, [150], [300], dict(window=70)),
    "softcap": (4, 2, 64, F16, F32, 16, [10, 1], [90, 64], dict(softcap=3.0)),
    "softcap_prompt": (4, 2, 128, BF16, BF16, 16, [80], [130], dict(softcap=20.0)),
    "sinks": (4, 2, 64, BF16, F32, 16, [10, 1], [90, 64], dict(sinks=True)),
    "sinks_prompt": (4, 2, 64, F16, F16, 16, [90], [90], dict(sinks=True, window=20)),
    "peaked": (4, 2, 128, BF16, F32, 16, [5, 70], [300, 70], dict(peak=6.0)),
    "peaked_f16": (4, 2, 128, F16, F32, 16, [5, 70], [300, 70], dict(peak=6.0)),
    "more_tokens_than_positions": (2, 1, 64, BF16, F32, 16, [5, 3], [2, 0], {}),
    # windows that p - window would carry past -2^31, where a tile begins before the first position
    "more_tokens_widest_window": (2, 1, 64, BF16, F32, 16, [5, 3, 1], [2, 0, 1], dict(window=2 ** 31 - 1)),
    "more_tokens_widest_window_tiles": (2, 1, 64, BF16, BF16, 16, [70, 90], [30, 80], dict(window=2 ** 31 - 1)),
    "more_tokens_window": (2, 1, 64, F32, F32, 16, [70, 9], [30, 4], dict(window=3)),
    "softcap_wide": (4, 2, 64, F32, F32, 16, [3, 80], [90, 130], dict(softcap=50.0)),
    # pages that split a load's rows, and every width the prompt kernels compute at
    "prompt_pages_of_1": (4, 2, 128, BF16, BF16, 1, [70, 40], [130, 41], {}),
    "prompt_pages_of_5": (2, 1, 64, F16, F32, 5, [150], [333], {}),
    "prompt_pages_of_6_wide": (2, 1, 256, BF16, F32, 6, [70], [97], {}),
    "prompt_pages_of_12_wide": (2, 1, 248, F16, F16, 12, [70, 64], [97, 64], {}),
    "prompt_88": (3, 3, 88, BF16, F32, 24, [65, 66], [100, 66], dict(window=64)),
    "prompt_112": (2, 1, 112, F16, F16, 16, [129], [129], {}),
    "prompt_f32_wide": (2, 2, 200, F32, F32, 16, [129, 30], [140, 31], {}),
    "prompt_f32_pages_of_7": (1, 1, 128, F32, F32, 7, [129], [200], {}),
    "prompt_f32_64": (2, 1, 64, F32, F32, 16, [90], [300], {}),
    "split_tiles": (2, 1, 64, BF16, F32, 16, [70], [4100], {}),
    "split_tiles_f32": (1, 1, 32, F32, F32, 16, [70], [2100], dict(window=1999)),
    "split_tiles_f32_finer": (2, 1, 64, F32, F32, 16, [80, 40], [5200, 300], {}),
    "split_window_one_token": (8, 2, 64, BF16, F32, 16, [1, 1, 1], [5000, 4097, 3], dict(window=600)),
    "split_window_tiles": (4, 1, 64, BF16, BF16, 16, [40, 3], [5000, 700], dict(window=700)),
    "split_window_tiles_f32": (2, 1, 64, F32, F32, 24, [90, 33], [5000, 1600], dict(window=1500)),
    "split_window_of_one": (4, 1, 64, F16, F32, 16, [1, 2], [900, 901], dict(window=1)),
    "one_row_of_a_tile_more": (1, 1, 128, BF16, BF16, 16, [129, 257], [129, 300], {}),
    "negative_scale": (4, 2, 64, BF16, F32, 16, [1, 70], [90, 70], dict(scale=-0.2)),
    "no_scale": (4, 2, 64, F16, F32, 16, [1, 70], [90, 70], dict(scale=0.0)),
    "rising_scores": (2, 1, 64, F16, F32, 16, [3, 40], [700, 400], dict(rise=True)),
    "rising_scores_bf16": (2, 1, 128, BF16, BF16, 16, [3, 40], [700, 400], dict(rise=True)),
    "many_sequences": (2, 1, 32, F32, F32, 8, [1 + i % 2 for i in range(140)], [2 + i % 50 for i in range(140)], {}),
}


def attention_case(name):
    H, G, D, tc, tout, ps, counts, lengths, options = ATTENTION[name]
    options = dict(options)
    peak = options.pop("peak", 1.0)
    P = ref.Paged(counts, [max(n, 0) for n in lengths], G, D, ps, tc, 17, by_head=len(counts) % 2 == 0,
                  pad=8 if D % 16 else 0)
    q = (torch.randn(P.tokens, H, D, generator=P.g) * peak).to(tc)
    if options.pop("rise", False):  # scores that grow along the sequence, so that every tile brings a new maximum
        for i, n in enumerate(P.lengths):
            j = torch.arange(n)
            at = P.table[i].long()[j // ps], j % ps
            P.pools[0][1][at] = (P.pools[0][1][at].float() * 0.1 + j[:, None, None] * 0.05).to(tc)
        q = (0.5 + torch.rand(q.shape, generator=P.g)).to(tc)
    if options.get("sinks"):
        options["sinks"] = torch.randn(H, generator=P.g) * 2
    return P, q, tout, options


def check_attention(P, q, got, options, tout, scale):
    D = q.shape[2]
    for i, (rows, out, spread, size) in enumerate(ref.attention(P, q, scale, **options)):
        n = max(P.lengths[i], 1)
        weight = 2 * U * (D + 8) * size + U * (n + 64)
        if tout != F32:
            weight = weight + ref.bound_of(tout)
        tol = weight * spread + ref.half_step(tout, out.abs() + weight * spread)
        off = (got[rows].double() - out).abs() - tol
        assert (off <= 0).all(), f"sequence {i}: {off.max()} beyond the bound, rows {(off > 0).nonzero()[:4].tolist()}"


@pytest.mark.parametrize("name", list(ATTENTION))
def test_attention_paged(gpu, name):
    P, q, tout, options = attention_case(name)
    H, D = q.shape[1:]
    cache, batch = P.on(gpu)
    # rows of a wider matrix, with poison between them
    qd = torch.full((P.tokens, H * D + 16), float("nan"), dtype=q.dtype, device=gpu)
    qd[:, :H * D] = q.reshape(P.tokens, -1).to(gpu)
    out = torch.full((P.tokens, H * D + 8), 7.0, dtype=tout, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    on_gpu = {k: to(gpu, v) if torch.is_tensor(v) else v for k, v in options.items()}
    sv.attention(cache, batch, qd[:, :H * D].unflatten(1, (H, D)), out[:, :H * D].unflatten(1, (H, D)), ws, **on_gpu)
    assert sv.status(ws) == 0
    got = out.cpu()
    assert (got[P.starts[-1]:] == 7.0).all() and (got[:, H * D:] == 7.0).all()
    scale = options.pop("scale", 1.0 / math.sqrt(D))
    check_attention(P, q, got[:, :H * D].unflatten(1, (H, D)), options, tout, scale)


@pytest.mark.parametrize("name", ["decode", "decode_wide_f32", "decode_mqa", "few_tokens", "window", "sinks", "window_f32",
                                  "more_tokens_than_positions", "many_sequences"])
@pytest.mark.parametrize("loose", [dict(max_new=400), dict(tokens=700), dict(max_new=90, tokens=100000)])
def test_attention_paged_with_loose_bounds(gpu, name, loose):
    """Bounds above what the batch holds choose other kernels and splits, not other
    results; rows that the arrays do not reach are left alone."""
    P, q, tout, options = attention_case(name)
    H, D = q.shape[1:]
    cache, batch = P.on(gpu)
    tokens = max(loose.get("tokens", 0), P.tokens)
    batch = sv.Batch(batch.starts, batch.lengths, batch.table, tokens, max(loose.get("max_new", 0), P.max_new))
    qd = torch.full((tokens, H, D), float("nan"), dtype=q.dtype, device=gpu)
    qd[:P.starts[-1]] = q[:P.starts[-1]].to(gpu)
    out = torch.full((tokens, H, D), 7.0, dtype=tout, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    on_gpu = {k: to(gpu, v) if torch.is_tensor(v) else v for k, v in options.items()}
    sv.attention(cache, batch, qd, out, ws, **on_gpu)
    assert sv.status(ws) == 0
    assert (out[P.starts[-1]:] == 7.0).all()
    check_attention(P, q, out[:P.tokens].cpu(), options, tout, 1.0 / math.sqrt(D))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("counts,window", [([40], 0), ([4], 0), ([40], 12), ([150], 40), ([150], 0)])
def test_attention_paged_unseen_values_stay_out(gpu, dtype, counts, window):
    """NaN and infinities at positions that some rows of a tile see and others do
    not: the rows that do not are the bits they are without them."""
    H, G, D, L = 4, 2, 64, 160
    P = ref.Paged(counts, [L], G, D, 16, dtype, 23)
    q = torch.randn(P.tokens, H, D, generator=P.g).to(dtype)

    def run():
        cache, batch = P.on(gpu)
        out = torch.zeros(P.tokens, H, D, device=gpu)
        ws = sv.attention_workspace(cache, batch, H)
        sv.attention(cache, batch, q.to(gpu), out, ws, window=window)
        assert sv.status(ws) == 0
        return out.cpu()

    clean = run()
    n = counts[0]
    marks = {L - n // 2: float("nan"), L - 2: float("inf"), L - n + 1: float("-inf")}
    at = P.table[0].long()
    for j, value in marks.items():
        P.pools[1][1][at[j // 16], j % 16, :, 3] = value
    marked = run()
    for r in range(n):
        p = L - n + r
        seen = [v for j, v in marks.items() if j <= p and (not window or j > p - window)]
        same = marked[r] == clean[r]
        assert same[:, [d for d in range(D) if d != 3]].all(), r
        if not seen:
            assert same.all(), r
        else:
            assert not marked[r, :, 3].isfinite().any(), r
    # a NaN key spoils exactly the rows that see it
    j = L - n // 2
    P.pools[0][1][at[j // 16], j % 16, :, 5] = float("nan")
    spoiled = run()
    for r in range(n):
        p = L - n + r
        sees = j <= p and (not window or j > p - window)
        rest = spoiled[r][:, [d for d in range(D) if d != 3]].isnan()
        assert rest.all() if sees else not rest.any(), r


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("counts,lengths", [([1, 1], [1, 5]), ([1, 2], [3000, 9]), ([150, 40], [150, 3000])])
def test_attention_paged_scores_that_are_no_numbers(gpu, counts, lengths, dtype, sinks):
    """Sequence 0 sees nothing but scores of NaN, or of -inf: its rows are NaN, as a
    softmax over those is; a sink beside -inf alone takes all the weight. Sequence
    1 keeps its values."""
    H, G, D = 4, 2, 80
    P = ref.Paged(counts, lengths, G, D, 16, dtype, 6)
    cache, batch = P.on(gpu)
    q = torch.rand(P.tokens, H, D, generator=P.g).add_(0.5).to(dtype).to(gpu)
    sink = torch.zeros(H, device=gpu) if sinks else None
    ws = sv.attention_workspace(cache, batch, H)
    out = torch.empty(P.tokens, H, D, dtype=F32, device=gpu)
    sv.attention(cache, batch, q, out, ws, sinks=sink)
    want = out.cpu()[counts[0]:P.starts[-1]]
    assert torch.isfinite(want).all()
    mine = torch.tensor(P.pages[0], device=gpu)
    for value in (math.nan, -math.inf):
        cache.k[mine] = value
        sv.attention(cache, batch, q, out, ws, sinks=sink)
        got = out.cpu()
        if sinks and value < 0:
            assert (got[:counts[0]] == 0).all()
        else:
            assert torch.isnan(got[:counts[0]]).all()
        assert torch.equal(got[counts[0]:P.starts[-1]], want)
    assert sv.status(ws) == 0


def test_attention_paged_reports_what_it_does_not_follow(gpu):
    def run(change):
        P = ref.Paged([1, 2, 1], [40, 30, 20], 1, 32, 8, F32, 29)
        q = torch.randn(P.tokens, 2, 32, generator=P.g)
        want = [out for _, out, _, _ in ref.attention(P, q, 0.5)]
        change(P)
        cache, batch = P.on(gpu)
        out = torch.full((P.tokens, 2, 32), 7.0, device=gpu)
        ws = sv.attention_workspace(cache, batch, 2)
        sv.attention(cache, batch, q.to(gpu), out, ws, scale=0.5)
        st = sv.status(ws)
        assert (out[4:] == 7.0).all()
        return st, (out[0].cpu().double() - want[0][0]).abs().max() < 1e-4, (out[3].cpu().double() - want[2][0]).abs().max() < 1e-4

    def page(P):
        P.table[1, 2] = 10 ** 6

    def long(P):
        P.lengths = [40, 10 ** 6, 20]

    def many(P):
        P.max_new = 1

    assert run(lambda P: None) == (0, True, True)
    for change in (page, long, many):
        assert run(change) == (1, True, True)


@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("length,status", [(2 ** 31 - 2 ** 16 + 1, 1), (2 ** 31 - 1, 1)])
def test_paged_lengths_that_pass_31_bits(gpu, count, length, status):
    """Lengths near 2^31, which a table of 32768 pages of 65536 would cover: past the
    last one allowed they are reported and not followed, by the cache write either."""
    D, ps = 8, 65536
    pool = torch.zeros(1, ps, 1, D, dtype=F16, device=gpu)
    cache = sv.Cache.of(pool, torch.zeros_like(pool))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    table = torch.zeros(2, 32768, dtype=torch.int32, device=gpu)
    batch = sv.Batch(i32(0, count, count + 1), i32(length, 5), table, count + 1, count)
    q = torch.ones(count + 1, 1, D, dtype=F16, device=gpu)
    out = torch.full((count + 1, 1, D), 7.0, dtype=F16, device=gpu)
    ws = sv.attention_workspace(cache, batch, 1)
    rope = sv.Rope(D, device=gpu)
    cache.v[0, :5] = 2.0
    sv.attention(cache, batch, q, out, ws)
    assert sv.status(ws) == status
    assert (out[count] == 2.0).all() and (out[:count] == 7.0).all()
    cache.k.zero_()
    sv.rope_append(cache, batch, rope, q, q, q, out, ws)
    assert sv.status(ws) == status
    assert (cache.k[0, 4] != 0).any() and (cache.k[0, 5:] == 0).all() and (cache.k[0, :4] == 0).all()


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16), (F32, F32)])
def test_attention_paged_long(gpu, dtype, out):
    """Long sequences, whose keys go to hundreds of workgroups, beside short ones,
    single tokens and a chunk, against float64 on the GPU."""
    H, G, D, ps = 4, 2, 64, 16
    for counts, lengths in (([1, 1, 1], [70000, 5, 33001]), ([1, 40, 2], [20000, 30011, 17])):
        P = ref.Paged(counts, lengths, G, D, ps, dtype, 53)
        q = torch.randn(P.tokens, H, D, generator=P.g).to(dtype)
        cache, batch = P.on(gpu)
        got = torch.full((P.tokens, H, D), 7.0, dtype=out, device=gpu)
        ws = sv.attention_workspace(cache, batch, H)
        sv.attention(cache, batch, q.to(gpu), got, ws)
        assert sv.status(ws) == 0
        for i, (n, length) in enumerate(zip(counts, lengths)):
            k, v = (P.rows(i, w).to(gpu).double() for w in (0, 1))
            rows = slice(P.starts[i], P.starts[i] + n)
            hidden = torch.arange(length, device=gpu) > length - n + torch.arange(n, device=gpu)[:, None]
            for h in range(H):
                kk, vv, qq = k[:, h // (H // G)], v[:, h // (H // G)], q[rows, h].to(gpu).double()
                p = torch.softmax((qq @ kk.t() / math.sqrt(D)).masked_fill(hidden, -math.inf), 1)
                want, spread = p @ vv, p @ vv.abs()
                size = (qq.abs() @ kk.abs().t()).amax(1, keepdim=True) / math.sqrt(D)
                # (the sums of the n weights lie in pieces of at most 2000, joined in f32)
                weight = 2 * U * (D + 8) * size + U * (2000 + 600) + (0 if out == F32 else ref.bound_of(out))
                tol = weight * spread + ref.half_step(out, want.abs() + weight * spread)
                assert ((got[rows, h].double() - want).abs() <= tol).all(), (i, h)


def test_attention_paged_one_workspace_for_two_captures(gpu):
    """Two captured calls of different shapes that share a workspace, replayed one
    after the other in both orders."""
    calls = []
    need = 0
    for i, (counts, lengths) in enumerate((([1, 1], [3000, 100]), ([50], [1300]))):
        P = ref.Paged(counts, lengths, 2, 64, 16, BF16, 60 + i)
        cache, batch = P.on(gpu)
        q = torch.randn(P.tokens, 8, 64, generator=P.g).to(BF16).to(gpu)
        need = max(need, sv.attention_workspace(cache, batch, 8).numel())
        calls.append((cache, batch, q, torch.zeros(P.tokens, 8, 64, device=gpu)))
    ws = sv.workspace(need, gpu)
    wants, graphs = [], []
    for cache, batch, q, out in calls:
        sv.attention(cache, batch, q, out, ws)
        torch.cuda.synchronize()
        wants.append(out.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sv.attention(cache, batch, q, out, ws)
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for c in calls:
            c[3].zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for c, want in zip(calls, wants):
            assert torch.equal(c[3], want), order
    assert sv.status(ws) == 0


def test_attention_paged_beyond_32_bit_offsets(gpu):
    """Pages more than 2^32 elements into the pool."""
    H, D, ps = 2, 128, 64
    pages = (1 << 32) // (ps * D) + 9
    k = torch.empty(pages, ps, 1, D, dtype=BF16, device=gpu)  # 8.6 GB each, most of it never touched
    v = torch.empty(pages, ps, 1, D, dtype=BF16, device=gpu)
    P = ref.Paged([1, 3], [100, 150], 1, D, ps, BF16, 31)
    q = torch.randn(P.tokens, H, D, generator=P.g).to(BF16)
    top = pages - P.pools[0][0].shape[0]
    for (_, view), pool in zip(P.pools, (k, v)):
        pool[top:] = view.to(gpu)
    _, batch = P.on(gpu)
    table = torch.where(P.table >= 0, P.table + top, P.table).to(gpu)
    batch = sv.Batch(batch.starts, batch.lengths, table, P.tokens, P.max_new)
    cache = sv.Cache.of(k, v)
    rope = sv.Rope(D, device=gpu)
    out = torch.zeros(P.tokens, H, D, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    sv.attention(cache, batch, q.to(gpu), out, ws)
    check_attention(P, q, out.cpu(), {}, F32, 1.0 / math.sqrt(D))
    x = torch.randn(P.tokens, H + 2, D, generator=P.g)
    xd = x.to(gpu)
    qo = torch.zeros(P.tokens, H, D, dtype=BF16, device=gpu)
    sv.rope_append(cache, batch, rope, xd[:, :H], xd[:, H:H + 1], xd[:, H + 1:], qo, ws)
    assert sv.status(ws) == 0
    last = int(table[1, 149 // ps])
    assert torch.equal(v[last, 149 % ps, 0].cpu(), x[3, H + 1].to(BF16))


def test_attention_paged_captured_and_replayed(gpu):
    """A captured step (cache write and attention) follows the lengths, tables and
    rows its arrays hold at each replay, with eager calls between replays."""
    H, G, D, ps, B, cap = 8, 2, 64, 16, 3, 40
    pool = [torch.zeros(B * cap, ps, G, D, dtype=BF16, device=gpu) for _ in range(2)]
    cache = sv.Cache.of(*pool)
    table = torch.randperm(B * cap, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(B, cap).to(gpu)
    starts = torch.arange(B + 1, dtype=torch.int32, device=gpu)
    lengths = torch.tensor([1, 200, 37], dtype=torch.int32, device=gpu)
    batch = sv.Batch(starts, lengths, table, B, 1)
    rope = sv.Rope(D, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(2)
    for t in pool:
        t.normal_(generator=g)
    x = torch.randn(B, H + 2 * G, D, generator=g, device=gpu)
    qr = torch.zeros(B, H, D, dtype=BF16, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    eager_ws = sv.attention_workspace(cache, batch, H)

    def step(out, ws):
        sv.rope_append(cache, batch, rope, x[:, :H], x[:, H:H + G], x[:, H + G:], qr, ws)
        sv.attention(cache, batch, qr, out, ws)

    out, eager = torch.zeros(B, H, D, device=gpu), torch.zeros(B, H, D, device=gpu)
    step(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws)
    for replay in range(8):
        lengths.add_(torch.tensor([1, 50, 3], dtype=torch.int32, device=gpu))
        x.normal_(generator=g)
        if replay == 4:
            table.copy_(table.flip(0))
        step(eager, eager_ws)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), replay
        assert (out != 0).any()
    assert sv.status(ws) == 0 and sv.status(eager_ws) == 0


def test_attention_paged_calls_in_flight(gpu):
    """Calls on streams of their own, each with its workspace, leave each other alone."""
    calls = []
    for i in range(8):
        P = ref.Paged([1, 1 + i % 3 * 20], [700 + i, 100 + i], 2, 64, 16, BF16, 40 + i)
        q = torch.randn(P.tokens, 8, 64, generator=P.g).to(BF16).to(gpu)
        cache, batch = P.on(gpu)
        out = torch.zeros(P.tokens, 8, 64, device=gpu)
        ws = sv.attention_workspace(cache, batch, 8)
        sv.attention(cache, batch, q, out, ws)
        calls.append((cache, batch, q, out.clone(), torch.zeros_like(out), ws, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(4):
        for cache, batch, q, want, out, ws, stream in calls:
            out.zero_()
        torch.cuda.synchronize()
        for cache, batch, q, want, out, ws, stream in calls:
            sv.attention(cache, batch, q, out, ws, stream=stream)
        torch.cuda.synchronize()
        for cache, batch, q, want, out, ws, stream in calls:
            assert torch.equal(out, want)


# ---------------------------------------------------------------- sampling --

def f32(x):
    return float(np.float32(x))


def light_error(x, temperature, chosen, p):
    """Relative error of the mass kept, beyond its steps of 2^-44 of the largest
    weight. Weights from 1/8 on come from double arithmetic; a smaller one, w = 2^t,
    from a float t that carries two roundings of 2^-24 of itself (the difference of
    logits, the product) and an exponential good to a unit in the last place: w
    times (2 |t| ln 2 + 2) 2^-24. These add up over the light weights at worst (1/7:
    the border is itself a float), against the mass kept, which is the chosen one's
    weight over its probability."""
    if temperature == 0.0:
        return 0.0
    x = x.double()
    t = torch.where(x == -math.inf, -math.inf, (x - x.max()) / f32(temperature)) / math.log(2.0)
    w = torch.exp2(t)
    light = (w < 1 / 7) & (t > -47)
    return float((w[light] * (2 * t[light].abs() * math.log(2.0) + 2)).sum()) * U * p / float(w[chosen])


def check_sample(gpu, x, uniform, stride=None, **settings):
    rows, vocab = x.shape
    xd = torch.full((rows, stride or vocab), 1e30, device=gpu)
    xd[:, :vocab] = x.to(gpu)
    kinds = dict(temperature=F32, top_k=torch.int32, top_p=F32, min_p=F32)
    on = {k: torch.tensor(v, dtype=kinds[k], device=gpu) for k, v in settings.items()}
    u = torch.tensor(uniform, dtype=F32, device=gpu)
    ws = sv.workspace(fmx.lib().fmx_sample_workspace_bytes(rows, vocab), gpu)
    ids, probs = sv.sample(xd[:, :vocab], u, ws, **on)
    assert sv.status(ws) == 0
    ids, probs = ids.cpu().tolist(), probs.cpu().tolist()
    for r in range(rows):
        want, p = ref.sample(x[r], f32(uniform[r]), **{k: (f32(v[r]) if k != "top_k" else v[r]) for k, v in settings.items()})
        assert ids[r] == want, (r, {k: v[r] for k, v in settings.items()})
        assert abs(probs[r] - p) <= p * (U + light_error(x[r], settings.get("temperature", [1.0] * rows)[r], want, p)) \
            + vocab * 2.0 ** -44, r


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8192, 8193, 32000, 32769, 131072, 262144])
@pytest.mark.parametrize("settings", ["plain", "top_k", "top_p", "min_p", "all"])
def test_sample(gpu, vocab, settings):
    rows = 12
    g = torch.Generator().manual_seed(vocab + len(settings))
    x = torch.randn(rows, vocab, generator=g) * 2
    x[:, :: max(1, vocab // 20)] += torch.rand(rows, len(range(0, vocab, max(1, vocab // 20))), generator=g) * 12
    u = torch.rand(rows, generator=g).tolist()
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    s = dict(temperature=[0.0, 0.05, 100.0] + (0.4 + torch.rand(rows - 3, generator=g)).tolist())
    if settings in ("top_k", "all"):
        s["top_k"] = [0, 1, 2, 5000] + torch.randint(1, 300, (rows - 4,), generator=g).tolist()
    if settings in ("top_p", "all"):
        s["top_p"] = [0.0, 1.0, 2.0, 0.999] + torch.rand(rows - 4, generator=g).tolist()
    if settings in ("min_p", "all"):
        s["min_p"] = [0.0, 1.0, 0.5, -1.0] + (torch.rand(rows - 4, generator=g) * 0.2).tolist()
    check_sample(gpu, x, u, stride=vocab + 3, **s)


@pytest.mark.parametrize("vocab", [5, 3000, 20000, 100001])
def test_sample_ties_and_masks(gpu, vocab):
    """All logits equal, a few values only, masks of -inf and of the type's lowest
    value, zeros of both signs: equal ones in the order of their ids."""
    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(F32).min
    x = torch.stack([
        torch.zeros(vocab),
        torch.randint(0, 3, (vocab,), generator=g).float(),
        torch.where(torch.rand(vocab, generator=g) < 0.5, -math.inf, 1.0),
        torch.full((vocab,), low),
        torch.where(torch.arange(vocab) == vocab // 2, 0.0, -math.inf),
        torch.where(torch.rand(vocab, generator=g) < 0.9, low, torch.randn(vocab, generator=g)),
        torch.where(torch.rand(vocab, generator=g) < 0.5, -0.0, 0.0),
        3.0 + torch.randint(0, 4000, (vocab,), generator=g) * 2.0 ** -20,
        torch.linspace(-1.7e38, 1.7e38, vocab),  # (a wider one's step is infinite, and the row refused)
        torch.where(torch.rand(vocab, generator=g) < 0.5, 1e-42, 0.0),
    ])
    rows = x.shape[0]
    for k, u in ((0, 0.5), (3, 0.999), (vocab // 2 + 1, 0.75), (vocab, 0.25)):
        check_sample(gpu, x, [u] * rows, top_k=[k] * rows, temperature=[1.0] * rows)
    check_sample(gpu, x, [0.625] * rows, top_p=[0.5] * rows)
    check_sample(gpu, x, [0.125] * rows, min_p=[1.0] * rows, temperature=[2.0] * rows)
    check_sample(gpu, x, [0.875] * rows, temperature=[math.inf] * rows)
    check_sample(gpu, x, [0.875] * rows, temperature=[1e-45] * rows)


@pytest.mark.parametrize("crowd", [31, 33, 64, 65, 400, 511, 513, 1000, 1025, 1500])
def test_sample_crowds_within_a_step(gpu, crowd):
    """`crowd` logits that share one of the search's steps, equal or a few last
    places apart, among 6000 of which the largest is far above: the choice, the
    end of top-p and of a large top-k fall among them. The largest weighs 1 and
    the crowd's members 2^-8 of that (their differences are below 2^-20): the
    distribution's halves and quarters lie inside."""
    vocab, g = 6000, torch.Generator().manual_seed(crowd)
    rows = []
    for spread in (0.0, 2.0 ** -19, 2.0 ** -17):
        x = torch.full((vocab,), -20.0) - torch.rand(vocab, generator=g) * 5
        ids = torch.randperm(vocab, generator=g)
        at = 4.0 - 8 * math.log(2.0)
        x[ids[:crowd]] = at + torch.randint(0, 8, (crowd,), generator=g) * spread
        x[ids[crowd]] = 4.0
        rows.append(x)
    x = torch.stack(rows).repeat(3, 1)
    n = x.shape[0]
    u = [0.97, 0.6, 0.3, 0.9, 0.999, 0.5, 0.85, 0.7, 0.99]
    check_sample(gpu, x, u)
    check_sample(gpu, x, u, top_p=[0.9, 0.8, 0.55, 0.99, 0.7, 0.85, 0.6, 0.95, 0.75])
    check_sample(gpu, x, u, top_k=[300, 257, 999, 20, 30, 1000, 260, 5000, 100])
    check_sample(gpu, x, u, top_k=[crowd + 1, crowd, crowd // 2 + 1] * 3, top_p=[0.9] * n, min_p=[2.0 ** -8 - 2.0 ** -12] * n)


@pytest.mark.parametrize("vocab", [1, 700, 1500, 3000, 9001])
def test_sample_many_rows(gpu, vocab):
    """Enough rows for two smaller workgroups a CU: every setting at once, and rows
    of few values, whose crowds pass what such a workgroup lists."""
    rows, g = 520, torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g) * 2
    x[::5] = torch.randint(0, 3, (len(range(0, rows, 5)), vocab), generator=g).float()
    pick = lambda *values: [values[int(i)] for i in torch.randint(0, len(values), (rows,), generator=g)]
    u = torch.rand(rows, generator=g).tolist()
    check_sample(gpu, x, u, stride=vocab + 1)
    check_sample(gpu, x, u, temperature=pick(0.0, 0.5, 0.9, 1.7), top_k=pick(0, 1, 40, 256, 257, 2000),
                 top_p=pick(1.0, 0.9, 0.5), min_p=pick(0.0, 0.05))


@pytest.mark.parametrize("temperature", [1e-38, 1e-20, 2.0 ** -7, 33.0, 1e10, 3e38])
def test_sample_at_extreme_temperatures(gpu, temperature):
    """Weights that are all alike, or but one or two: the filters as ever. Alike
    weights (the last two) are 1 to the last place, so that their prefixes end
    where the counts say; u and top_p are odd multiples of 2^-13, never at an
    element's edge of the 1000 or 5000."""
    g = torch.Generator().manual_seed(3)
    for vocab in (1000, 5000):
        x = torch.randint(-40, 40, (4, vocab), generator=g) * 0.25
        u = [1.0 / 8192, 4095.0 / 8192, 8191.0 / 8192, 2047.0 / 8192]
        t = [temperature] * 4
        check_sample(gpu, x, u, temperature=t)
        check_sample(gpu, x, u, temperature=t, top_k=[1, 7, 300, 700])
        check_sample(gpu, x, u, temperature=t, top_p=[4097.0 / 8192] * 4, top_k=[0, 0, 500, 100])


def test_sample_refuses_rows_without_a_distribution(gpu):
    vocab = 1000
    x = torch.randn(7, vocab)
    x[0, 3] = math.nan
    x[1, 999] = math.inf
    x[2] = -math.inf
    t = torch.ones(7)
    t[3] = -1.0
    t[4] = math.nan
    u = torch.full((7,), 0.5)
    u[5] = math.nan
    ws = sv.workspace(fmx.lib().fmx_sample_workspace_bytes(7, vocab), gpu)
    ids, probs = sv.sample(x.to(gpu), u.to(gpu), ws, temperature=t.to(gpu))
    assert sv.status(ws) == 4
    assert ids.cpu().tolist()[:6] == [-1] * 6 and probs.cpu().tolist()[:6] == [0.0] * 6
    assert ids.cpu().tolist()[6] == ref.sample(x[6], 0.5)[0]


def test_sample_follows_the_distribution(gpu):
    """2^14 equally spaced uniforms give every token its share, within the one
    step either end of a token's stretch can take."""
    n, vocab = 1 << 14, 50
    x = torch.randn(1, vocab).expand(n, vocab)
    u = (torch.arange(n) + 0.5) / n
    ids, probs = sv.sample(x.contiguous().to(gpu), u.to(gpu))
    p = torch.softmax(x[0].double(), 0)
    count = torch.bincount(ids.cpu().long(), minlength=vocab).double() / n
    assert ((count - p).abs() <= 1.5 / n).all()
    assert ((probs.cpu().double() - p[ids.cpu().long()]).abs() <= 1e-7).all()


def test_sample_captured_and_replayed(gpu):
    rows, vocab = 5, 40000
    g = torch.Generator(device=gpu).manual_seed(8)
    x, u = torch.randn(rows, vocab, generator=g, device=gpu), torch.rand(rows, generator=g, device=gpu)
    top_p = torch.full((rows,), 0.9, device=gpu)
    ws = [sv.workspace(fmx.lib().fmx_sample_workspace_bytes(rows, vocab), gpu) for _ in range(2)]
    out = [(torch.zeros(rows, dtype=torch.int32, device=gpu), torch.zeros(rows, device=gpu)) for _ in range(2)]

    def run(i):
        sv.sample(x, u, ws[i], top_p=top_p, ids=out[i][0], probs=out[i][1])

    run(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(0)
    for replay in range(6):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        run(1)
        out[0][0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1]), replay
