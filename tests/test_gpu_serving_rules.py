"""What the serving operators promise beside their values, on an MI355X: how far
a 16-bit result may lie from the exact one, what may not change a token's bits,
which entries of a page table are read, on which stream a call's own tensors are
made."""
import math

import pytest
import torch

import serving_ref as ref
from freemoe_amd import fmx
from freemoe_amd import serving as sv

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,counts,lengths", [
    (8, 2, 128, [1, 1, 1], [5000, 300, 2]), (4, 4, 64, [1, 3, 16], [70, 900, 40]), (16, 1, 80, [1, 1], [1300, 64]),
    (2, 1, 256, [2, 8], [500, 8])])
def test_few_rows_are_rounded_once(gpu, dtype, heads, kv_heads, dim, counts, lengths):
    """Up to 16 rows of a sequence in 16 bits: the sums are those of an f32 result,
    and the one rounding is the output's. The bound is the f32 one (a score's D + 8
    roundings twice, n sums, some 64 for exponentials, scaling and the weights' last
    part) with half a step of the output; a weight in 16 bits alone would add half a
    step of sum_j p_j |v_j|."""
    P = ref.Paged(counts, lengths, kv_heads, dim, 16, dtype, 71)
    q = torch.randn(P.tokens, heads, dim, generator=P.g).to(dtype)
    cache, batch = P.on(gpu)
    out = torch.zeros(P.tokens, heads, dim, dtype=dtype, device=gpu)
    ws = sv.attention_workspace(cache, batch, heads)
    sv.attention(cache, batch, q.to(gpu), out, ws)
    assert sv.status(ws) == 0
    got = out.cpu().double()
    for i, (rows, want, spread, size) in enumerate(ref.attention(P, q, 1.0 / math.sqrt(dim))):
        error = (2 * U * (dim + 8) * size + U * (lengths[i] + 64)) * spread
        off = (got[rows] - want).abs() - error - ref.half_step(dtype, want.abs() + error)
        assert (off <= 0).all(), f"sequence {i}: {off.max()} beyond the bound, {int((off > 0).sum())} of {off.numel()}"


def test_sample_on_another_stream_with_its_own_tensors(gpu):
    """The current stream's memory is handed out again while its work still writes
    there: what a call on another stream makes for itself is not of that memory."""
    rows, vocab = 64, 20000
    g = torch.Generator(device=gpu).manual_seed(91)
    x, u = torch.randn(rows, vocab, generator=g, device=gpu), torch.rand(rows, generator=g, device=gpu)
    x[5, 7] = math.nan
    want = sv.sample(x, u)
    assert sv.status(want.ws) == 4 and want.ids[5] == -1 and want.probs[5] == 0
    side, a = torch.cuda.Stream(), torch.randn(4096, 4096, device=gpu)
    torch.cuda.synchronize()
    for _ in range(3):
        held = [torch.empty(rows, dtype=torch.int32, device=gpu) for _ in range(40)]
        for _ in range(8):
            a = a @ a * 1e-3  # some milliseconds
        for t in held:
            t.fill_(7)
        del held, t
        got = sv.sample(x, u, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got.ids, want.ids) and torch.equal(got.probs, want.probs)
        assert sv.status(got.ws, side) == 4 and sv.status(got.ws, side) == 0


def test_one_row_of_any_stride(gpu):
    """A tensor of one row has no stride to speak of: a slice of a row whose width
    no 16 bytes divide is taken."""
    H, G, D = 2, 1, 24
    P = ref.Paged([1], [30], G, D, 16, F32, 41, spare=0)
    wide = torch.randn(2, (H + 2 * G) * D + 3, generator=P.g)
    x = wide.to(gpu)[:, :(H + 2 * G) * D].unflatten(1, (H + 2 * G, D))[:1]
    cache, batch = P.on(gpu)
    rope, ws = sv.Rope(D, device=gpu), sv.attention_workspace(cache, batch, H)
    turned = torch.zeros(2, H * D + 1, device=gpu)[:, :H * D].unflatten(1, (H, D))[:1]
    sv.rope_append(cache, batch, rope, x[:, :H], x[:, H:H + G], x[:, H + G:], turned, ws)
    out = torch.zeros(2, H * D + 1, device=gpu)[:, :H * D].unflatten(1, (H, D))[:1]
    sv.attention(cache, batch, turned, out, ws)
    assert sv.status(ws) == 0
    same = torch.zeros(1, H, D, device=gpu)
    sv.attention(cache, batch, turned.contiguous(), same, ws)
    assert torch.equal(out, same) and (out != 0).any()
    want, size = ref.rope(wide[:1, :H * D].unflatten(1, (H, D)), torch.tensor([29]), rope.inv_freq.cpu(), 1.0, D, True)
    assert ((turned.cpu().double() - want).abs() <= 4 * U * size + U * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("softcap", [3.0, 50.0])
@pytest.mark.parametrize("counts", [[4], [40], [150]])
def test_softcap_of_unseen_keys_stays_out(gpu, dtype, counts, softcap):
    """Soft-capped scores of keys a token does not see, however large, and of other
    tokens' queries leave its bits alone: hidden keys, places behind the last one
    of its page, and the last token's query are made large in turn."""
    H, G, D, L, n = 4, 2, 64, 165, counts[0]
    P = ref.Paged(counts, [L], G, D, 16, dtype, 29)
    for pool, _ in P.pools:
        pool.nan_to_num_(0.01)
    # scores of about a twentieth of the cap, none near a quarter of it
    q = (torch.randn(P.tokens, H, D, generator=P.g) * 0.05 * softcap).to(dtype)
    at = P.table[0].long()

    def run():
        cache, batch = P.on(gpu)
        out = torch.zeros(P.tokens, H, D, device=gpu)
        ws = sv.attention_workspace(cache, batch, H)
        sv.attention(cache, batch, q.to(gpu), out, ws, softcap=softcap)
        assert sv.status(ws) == 0
        return out.cpu()

    clean = run()
    keys = P.pools[0][1]
    keys[at[L // 16], L % 16:] = 40.0  # behind the last position, in its page
    assert torch.equal(run()[:n], clean[:n])
    keys[at[(L - 1) // 16], (L - 1) % 16] = 40.0  # the last position: its own token sees it
    assert torch.equal(run()[:n - 1], clean[:n - 1])
    j = L - n // 2  # seen from token n - n // 2 on
    keys[at[j // 16], j % 16] = -40.0
    assert torch.equal(run()[:n - n // 2], clean[:n - n // 2])
    q[n - 1] = 40.0
    assert torch.equal(run()[:n - n // 2], clean[:n - n // 2])


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 12), (F16, 64, 1), (F32, 64, 3), (BF16, 256, 6), (F16, 128, 5),
                                            (F32, 96, 20), (BF16, 64, 16)])
@pytest.mark.parametrize("count,window", [(1, 20), (1, 1), (40, 33), (150, 50)])
def test_pages_before_the_window_are_not_read(gpu, dtype, dim, page, count, window):
    """A program that slides a window gives back the pages before it: their entries
    may hold anything, whatever the page size."""
    H, G, L = 4, 2, 333
    P = ref.Paged([count, 1], [L, 7], G, dim, page, dtype, 37)
    q = torch.randn(P.tokens, H, dim, generator=P.g).to(dtype)
    cache, batch = P.on(gpu)
    first = L - count - window + 1  # the first position any new token sees
    gone = first // page
    assert gone > 0
    batch.table[0, :gone] = torch.tensor([-1, 10 ** 6] * gone, dtype=torch.int32, device=gpu)[:gone]
    out = torch.zeros(P.tokens, H, dim, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    sv.attention(cache, batch, q.to(gpu), out, ws, window=window)
    assert sv.status(ws) == 0
    got = out.cpu().double()
    for i, (rows, want, spread, size) in enumerate(ref.attention(P, q, 1.0 / math.sqrt(dim), window=window)):
        error = (2 * U * (dim + 8) * size + U * (L + 64)) * spread
        assert ((got[rows] - want).abs() <= error + ref.half_step(F32, want.abs() + error)).all(), i


@pytest.mark.parametrize("scale,cap", [(0.125, 1e-30), (1e20, 1e-10), (0.0, 2.0 ** -126), (0.125, 2.0 ** 99), (-1e15, 4.0)])
@pytest.mark.parametrize("dtype,counts", [(F32, [5]), (BF16, [70])])
def test_extreme_softcaps(gpu, dtype, counts, scale, cap):
    """The smallest and largest caps a call takes, down to scores that all are 0 or
    plus and minus the cap (q . k = 0 stays 0 there)."""
    H, G, D, L = 2, 1, 64, 100
    P = ref.Paged(counts, [L], G, D, 16, dtype, 43)
    P.pools[0][1][P.table[0].long()[3], 2] = 0.0  # one key of zeros
    q = torch.randn(P.tokens, H, D, generator=P.g).to(dtype)
    cache, batch = P.on(gpu)
    out = torch.zeros(P.tokens, H, D, device=gpu)
    ws = sv.attention_workspace(cache, batch, H)
    sv.attention(cache, batch, q.to(gpu), out, ws, scale=scale, softcap=cap)
    assert sv.status(ws) == 0
    got = out.cpu().double()
    for rows, want, spread, size in ref.attention(P, q, scale, softcap=cap):
        # a score's error: the roundings of its dot and of the few steps behind it, which
        # the tangent passes on at most once; of a scale far above the cap the side q . k
        # lies on is all that counts, and what is left are the cap's own roundings
        score = (D + 16) * size if abs(scale) <= 1e9 * cap else 8 * cap
        error = (2 * U * score + U * (L + 64)) * spread
        assert ((got[rows] - want).abs() <= error + ref.half_step(F32, want.abs() + error)).all()


@pytest.mark.parametrize("rows,vocab", [(256, 3000), (257, 3000), (300, 9001), (511, 700), (512, 3000)])
def test_sampled_rows_do_not_depend_on_how_many_there_are(gpu, rows, vocab):
    """The number of rows chooses the workgroup: a row's id and probability are the
    bits they are in a small call."""
    g = torch.Generator(device=gpu).manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device=gpu) * 2
    x[::7] = torch.randint(0, 3, x[::7].shape, generator=g, device=gpu).float()
    u = torch.rand(rows, generator=g, device=gpu)
    settings = dict(temperature=0.5 + torch.rand(rows, generator=g, device=gpu),
                    top_k=torch.randint(0, 400, (rows,), generator=g, device=gpu).to(torch.int32),
                    top_p=0.6 + 0.5 * torch.rand(rows, generator=g, device=gpu),
                    min_p=0.05 * torch.rand(rows, generator=g, device=gpu))
    for names in ((), ("top_p",), ("temperature", "top_k"), tuple(settings)):
        some = {n: settings[n] for n in names}
        got = sv.sample(x, u, **some)
        assert sv.status(got.ws) == 0
        for at in range(0, rows, 50):
            few = sv.sample(x[at:at + 50], u[at:at + 50], **{n: t[at:at + 50] for n, t in some.items()})
            assert torch.equal(few.ids, got.ids[at:at + 50]) and torch.equal(few.probs, got.probs[at:at + 50]), (names, at)
