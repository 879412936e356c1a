"""Performance cases of the serving operators: rotary positions with the cache
write, attention over a paged cache, and sampling.

  rope       q and k rotated at their positions, k and v written into their
             sequences' pages
  attention  a ragged batch of new tokens (one each, or a prompt's chunk) over
             the pages their sequences hold
  sample     one token per row of logits, from given uniform numbers

`run` computes the plain form, torch operations in 32 bits (64 for angles and
probability sums) rounded once, or, where `own` is true, the calls of
freemoe_amd.fmx that a program makes.
"""
import ctypes
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _rope(name, **kw):
    case = dict(name=name, kind="rope", sequences=1, new=1, ragged=False, length=2000, heads=32, kv_heads=8,
                head_dim=128, dims=128, layout="half", scaling="none", source="f32", type="bf16", page_size=16,
                by_head=False)
    case.update(kw)
    return case


def _attention(name, **kw):
    case = dict(name=name, kind="attention", sequences=1, new=1, ragged=False, length=2000, heads=32, kv_heads=8,
                head_dim=128, type="bf16", out="f32", window=0, softcap=0.0, sinks=False, page_size=16, by_head=False)
    case.update(kw)
    return case


def listed():
    return [
        # one token of one conversation: all latency
        _rope("rope_one_token"),
        # a long prompt of one sequence, context extended eightfold
        _rope("rope_prompt_4096", new=4096, length=4096, scaling="yarn"),
        # a ragged batch of prompt chunks far into their sequences, part of each
        # head rotated in neighbouring pairs, an f32 cache
        _rope("rope_ragged_partial_f32", sequences=7, new=300, ragged=True, length=20000, heads=20, kv_heads=5,
              head_dim=96, dims=64, layout="interleaved", scaling="linear", type="f32"),
        # one token in the middle of a conversation, the cache in f32
        _attention("attention_one_token_f32_2000", type="f32"),
        # one token over a long document
        _attention("attention_one_token_131072", length=131072, type="f16", out="f16", page_size=64),
        # a serving batch's step: 64 sequences of very different lengths
        _attention("attention_64_tokens_ragged_8192", sequences=64, ragged=True, length=8192),
        # a prompt from its first token, in a 16-bit model
        _attention("attention_prompt_4096", new=4096, length=4096, out="bf16", page_size=32),
        # the last chunk of a long prompt: the largest call
        _attention("attention_chunk_2048_of_16384", new=2048, length=16384, out="bf16", page_size=64, by_head=True),
        # a ragged batch of prompts on f32 caches with a sliding window
        _attention("attention_ragged_window_f32", sequences=5, new=700, ragged=True, length=1800, heads=16, kv_heads=8,
                   head_dim=96, type="f32", window=1000, page_size=24),
        # one token's logits
        dict(name="sample_one_row_32000", kind="sample", rows=1, vocab=32000, mode="all"),
        # a serving batch over a large vocabulary
        dict(name="sample_64_rows_131072", kind="sample", rows=64, vocab=131072, mode="all"),
        # many rows, nucleus sampling alone
        dict(name="sample_512_rows_32001", kind="sample", rows=512, vocab=32001, mode="top_p"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


# What a drawn case may reach of the largest listed one.
MOST_PAIRS = 2048 * 16384 * 32 * 128  # query rows x positions x head width
MOST_CACHE = 64 * 8192 * 8 * 128      # cached positions x kv heads x head width


def _heads(rng):
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    return kv_heads * rng.choice([1, 2, 4, 8] if kv_heads < 16 else [1, 2]), kv_heads


def draw(rng):
    kind = rng.choice(["rope", "attention", "attention", "attention", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 500, 160000)
        return dict(kind=kind, rows=max(1, min(_log_int(rng, 1, 512), 64 * 131072 // vocab)), vocab=vocab,
                    mode=rng.choice(["all", "top_k", "top_p", "min_p", "plain"]))
    heads, kv_heads = _heads(rng)
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    case = dict(kind=kind, sequences=_log_int(rng, 1, 64), ragged=rng.random() < 0.7, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, type=rng.choice(["f32", "f16", "bf16", "bf16"]),
                page_size=rng.choice([1, 16, 16, 24, 32, 64, 128]), by_head=rng.random() < 0.3)
    if kind == "rope":
        case["sequences"] = min(case["sequences"], 16)
        case["new"] = _log_int(rng, 1, 4096 // case["sequences"])
        case["length"] = case["new"] + _log_int(rng, 1, 60000 // case["sequences"])
        case["dims"] = rng.choice([head_dim, head_dim, head_dim // 2, 32])
        case["layout"] = rng.choice(["half", "interleaved"])
        case["scaling"] = rng.choice(["none", "linear", "yarn"])
        case["source"] = rng.choice(["f32", "f32", case["type"]])
        return case
    case["length"] = min(_log_int(rng, 1, 65536), MOST_CACHE // (case["sequences"] * kv_heads * head_dim))
    case["new"] = 1
    if rng.random() < 0.6:  # chunks of a prompt, all of it at times
        most = min(4096, MOST_PAIRS // (case["sequences"] * heads * head_dim * case["length"]), case["length"])
        if case["type"] == "f32":
            most = min(most, max(1, MOST_PAIRS // 16 // (case["sequences"] * heads * head_dim * case["length"])))
        case["new"] = _log_int(rng, 1, max(1, most))
    case["out"] = rng.choice(["f32", case["type"]])
    case["window"] = rng.choice([0, 0, 0, _log_int(rng, 1, case["length"])])
    case["softcap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
    case["sinks"] = rng.random() < 0.2
    return case


# ------------------------------------------------------------------ inputs --

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _counts(case):
    """New tokens and lengths of each sequence: the same for every seed, so that
    every pass of a case does the same work."""
    B, new, length = case["sequences"], case["new"], case["length"]
    if not case["ragged"] or B == 1:
        return [new] * B, [max(new, length)] * B
    news, lengths = [], []
    for i in range(B):  # golden-ratio steps: spread evenly over the range, in no order
        f = (0.5 + i * 0.6180339887498949) % 1.0
        news.append(max(1, int(round(new * (0.25 + 0.75 * f)))) if i else new)
        lengths.append(max(news[-1], int(round(length * (0.02 + 0.98 * ((f * 7.0) % 1.0))))) if i else max(new, length))
    return news, lengths


def _inv_freq(dims, scaling):
    """Angles per position and the magnitude of the rotated pairs, base 10000,
    8 times the context of 4096 the angles were trained for."""
    base, factor, context = 10000.0, 8.0, 4096.0
    f = [base ** (-2.0 * c / dims) for c in range(dims // 2)]
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    if scaling == "yarn":
        def turns_at(n):
            return dims * math.log(context / (n * 2.0 * math.pi)) / (2.0 * math.log(base))

        low, high = max(0, math.floor(turns_at(32.0))), min(dims - 1, math.ceil(turns_at(1.0)))
        out = []
        for c, x in enumerate(f):
            ramp = min(1.0, max(0.0, (c - low) / max(high - low, 0.001)))
            out.append(x / factor * ramp + x * (1.0 - ramp))
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _pages(case, g, lengths):
    """The two pools, every value drawn (the places no token owns as well), and
    the table: the pages of a sequence lie anywhere in the pool."""
    ps, kvh, D = case["page_size"], case["kv_heads"], case["head_dim"]
    stride = max((n + ps - 1) // ps for n in lengths) + 1
    pages = sum((n + ps - 1) // ps for n in lengths) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), stride, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lengths):
        count = (n + ps - 1) // ps
        table[i, :count] = order[at:at + count]
        at += count
    shape = (pages, kvh, ps, D) if case["by_head"] else (pages, ps, kvh, D)
    k = torch.empty(shape, dtype=TYPES[case["type"]], device="cuda").normal_(generator=g)
    v = torch.empty(shape, dtype=TYPES[case["type"]], device="cuda").normal_(generator=g)
    return k, v, table


def _by_position(case, pool):
    """The pool as [page, place, kv head, element]."""
    return pool.transpose(1, 2) if case["by_head"] else pool


SPARE = 2  # rows behind the last sequence, as a padded batch has


def _paged(case, seed):
    g = _generator(seed)
    news, lengths = _counts(case)
    k, v, table = _pages(case, g, lengths)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    to = dict(dtype=torch.int32, device="cuda")
    return g, dict(case=dict(case), k=k, v=v, table=table, starts=torch.tensor(starts, **to),
                   lengths=torch.tensor(lengths, **to), tokens=starts[-1] + SPARE, max_new=max(news),
                   max_length=max(lengths),
                   workspace=torch.zeros(256, dtype=torch.uint8, device="cuda"))


def _prepare_rope(case, seed):
    g, s = _paged(case, seed)
    H, kvh, D, T = case["heads"], case["kv_heads"], case["head_dim"], s["tokens"]
    # one fused projection's rows
    s["qkv"] = _randn(g, T, (H + 2 * kvh) * D).to(TYPES[case["source"]])
    inv, s["magnitude"] = _inv_freq(case["dims"], case["scaling"])
    s["inv_freq"] = torch.tensor(inv, dtype=torch.float64, device="cuda")
    s["q_out"] = torch.zeros(T, H, D, dtype=TYPES[case["type"]], device="cuda")
    return s


def _prepare_attention(case, seed):
    g, s = _paged(case, seed)
    H, D, T = case["heads"], case["head_dim"], s["tokens"]
    s["q"] = _randn(g, T, H, D).to(TYPES[case["type"]])
    s["out"] = torch.zeros(T, H, D, dtype=TYPES[case["out"]], device="cuda")
    s["sinks"] = _randn(g, H) if case["sinks"] else None
    return s


def _prepare_sample(case, seed):
    g = _generator(seed)
    R, V, mode = case["rows"], case["vocab"], case["mode"]
    # a broad body and a few likely tokens, as a language model's logits have
    logits = 2.0 * _randn(g, R, V)
    few = min(V, 24)
    at = torch.randint(0, V, (R, few), generator=g, device="cuda")
    logits.scatter_add_(1, at, 12.0 * torch.rand(R, few, generator=g, device="cuda"))

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(R, generator=g, device="cuda")

    s = dict(case=dict(case), logits=logits, uniform=torch.rand(R, generator=g, device="cuda"),
             temperature=uniform(0.5, 1.3), top_k=None, top_p=None, min_p=None)
    if mode in ("all", "top_k"):
        s["top_k"] = torch.randint(1, 200, (R,), generator=g, device="cuda").to(torch.int32)
    if mode in ("all", "top_p"):
        s["top_p"] = uniform(0.7, 1.0)
    if mode in ("all", "min_p"):
        s["min_p"] = uniform(0.0, 0.1)
    s["ids"] = torch.zeros(R, dtype=torch.int32, device="cuda")
    s["probs"] = torch.zeros(R, device="cuda")
    return s


def prepare(case, seed):
    return {"rope": _prepare_rope, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, seed)


# --------------------------------------------------------------- plain form --

def _rows(s):
    """Sequence, place among its new tokens and position of every row, and
    whether a sequence owns it."""
    t = torch.arange(s["tokens"], device="cuda")
    starts = s["starts"].long()
    owned = t < starts[-1]
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp_max(starts.numel() - 2)
    place = t - starts[seq]
    position = s["lengths"].long()[seq] - (starts[seq + 1] - starts[seq]) + place
    return owned, seq, place, position


def _plain_rope(s):
    c = s["case"]
    H, kvh, D, R, ps, T = c["heads"], c["kv_heads"], c["head_dim"], c["dims"], c["page_size"], s["tokens"]
    owned, seq, _, position = _rows(s)
    x = s["qkv"].float().reshape(T, H + 2 * kvh, D)
    angle = position.double()[:, None] * s["inv_freq"]
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    rot = x[:, :H + kvh]
    if c["layout"] == "half":
        a, b = rot[..., :R // 2], rot[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos, rot[..., R:]), dim=-1)
    else:
        a, b = rot[..., 0:R:2], rot[..., 1:R:2]
        pair = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
        turned = torch.cat((pair, rot[..., R:]), dim=-1)
    s["q_out"].copy_(torch.where(owned[:, None, None], turned[:, :H].to(s["q_out"].dtype), s["q_out"]))
    n = T - SPARE  # (the rows behind the last sequence have no place in the table)
    at = (s["table"].long()[seq[:n], position[:n] // ps], position[:n] % ps)
    _by_position(c, s["k"])[at] = turned[:n, H:].to(s["k"].dtype)
    _by_position(c, s["v"])[at] = x[:n, H + kvh:].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    c = s["case"]
    H, kvh, D, ps, T = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"], s["tokens"]
    B, N, P, G = c["sequences"], s["max_new"], s["max_length"], H // kvh
    starts, lengths = s["starts"].long(), s["lengths"].long()
    owned, seq, place, _ = _rows(s)
    j = torch.arange(P, device="cuda")
    held = j[None, :] < lengths[:, None]
    page = torch.where(held, s["table"].long()[:, j // ps], 0)
    keys = _by_position(c, s["k"])[page, j % ps].float()  # [B, P, kv heads, D]
    values = torch.where(held[..., None, None], _by_position(c, s["v"])[page, j % ps].float(), 0.0)
    i = torch.arange(N, device="cuda")
    q = s["q"][(starts[:-1, None] + i).clamp_max(T - 1)].float()  # [B, N, H, D]
    q = q.reshape(B, N, kvh, G, D).permute(0, 2, 3, 1, 4).reshape(B, kvh, G * N, D)
    score = torch.matmul(q, keys.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
    if c["softcap"]:
        score = torch.tanh(score / c["softcap"]) * c["softcap"]
    position = (lengths - (starts[1:] - starts[:-1]))[:, None] + i  # [B, N]
    seen = (j <= position[..., None]) & held[:, None, :]
    if c["window"]:
        seen &= j > position[..., None] - c["window"]
    score = score.reshape(B, kvh, G, N, P).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    sink = None
    if s["sinks"] is not None:
        sink = s["sinks"].reshape(1, kvh, G, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    score = torch.exp(score - top)
    total = score.sum(dim=-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(score.reshape(B, kvh, G * N, P), values.permute(0, 2, 1, 3)).reshape(B, kvh, G, N, D)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, N, H, D)[seq, place.clamp(0, N - 1)]
    s["out"].copy_(torch.where(owned[:, None, None], out.to(s["out"].dtype), s["out"]))
    return s["out"]


def _plain_sample(s):
    x, V = s["logits"], s["case"]["vocab"]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x.double() - x[:, :1].double()) / s["temperature"].double()[:, None])
    mass = torch.cumsum(w, dim=1)
    count = torch.full((x.shape[0], 1), V, dtype=torch.int64, device="cuda")
    if s["top_k"] is not None:
        count = torch.minimum(count, s["top_k"].long()[:, None])
    if s["top_p"] is not None:
        least = s["top_p"].double()[:, None] * mass.gather(1, count - 1)
        count = torch.minimum(count, (mass < least).sum(dim=1, keepdim=True) + 1)
    if s["min_p"] is not None:
        count = torch.minimum(count, (w >= s["min_p"].double()[:, None]).sum(dim=1, keepdim=True))
    kept = mass.gather(1, count - 1)
    chosen = (mass <= s["uniform"].double()[:, None] * kept).sum(dim=1, keepdim=True)
    chosen = torch.minimum(chosen, count - 1)
    return {"ids": order.gather(1, chosen)[:, 0].to(torch.int32), "probs": (w.gather(1, chosen) / kept)[:, 0].float()}


# ------------------------------------------------------------- own operators --

def _descriptors(fmx, s):
    """The cache's and the batch's descriptors, which a program keeps."""
    c = s["case"]
    page, a, b = s["k"].stride()[:3]
    place, head = (b, a) if c["by_head"] else (a, b)
    cache = fmx.PagedCache(TYPE_IDS[c["type"]], c["kv_heads"], c["head_dim"], c["page_size"], s["k"].shape[0], page,
                           place, head, s["k"].data_ptr(), s["v"].data_ptr())
    batch = fmx.PagedBatch(c["sequences"], s["tokens"], s["max_new"], s["table"].shape[1], s["starts"].data_ptr(),
                           s["lengths"].data_ptr(), s["table"].data_ptr())
    return cache, batch


def _own_rope(s):
    from freemoe_amd import fmx
    c, qkv = s["case"], s["qkv"]
    if "held" not in s:
        rope = fmx.Rope(0 if c["layout"] == "interleaved" else 1, c["dims"], s["inv_freq"].data_ptr(),
                        s["magnitude"], None)
        s["held"] = (*_descriptors(fmx, s), rope)
    cache, batch, rope = s["held"]
    H, kvh, D, stride = c["heads"], c["kv_heads"], c["head_dim"], qkv.shape[1]
    q = qkv.data_ptr()
    k = q + H * D * BYTES[c["source"]]
    v = k + kvh * D * BYTES[c["source"]]
    fmx.call("fmx_rope_append", ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(rope), H,
             TYPE_IDS[c["source"]], q, stride, k, stride, v, stride, s["q_out"].data_ptr(), H * D,
             s["workspace"].data_ptr(), s["workspace"].numel(), fmx.stream_handle())
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attention(s):
    from freemoe_amd import fmx
    c = s["case"]
    H, D = c["heads"], c["head_dim"]
    if "held" not in s:
        cache, batch = _descriptors(fmx, s)
        options = fmx.AttentionOptions(1.0 / math.sqrt(D), c["softcap"], c["window"],
                                       None if s["sinks"] is None else s["sinks"].data_ptr())
        need = fmx.lib().fmx_attention_paged_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), H)
        s["held"] = (cache, batch, options, torch.zeros(need, dtype=torch.uint8, device="cuda"))
    cache, batch, options, workspace = s["held"]
    fmx.call("fmx_attention_paged", ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(options), H,
             s["q"].data_ptr(), H * D, TYPE_IDS[c["out"]], s["out"].data_ptr(), H * D, workspace.data_ptr(),
             workspace.numel(), fmx.stream_handle())
    return s["out"]


def _own_sample(s):
    from freemoe_amd import fmx
    c = s["case"]
    if "held" not in s:
        need = fmx.lib().fmx_sample_workspace_bytes(c["rows"], c["vocab"])
        s["held"] = (fmx.Sampling(*(None if s[n] is None else s[n].data_ptr()
                                    for n in ("temperature", "top_k", "top_p", "min_p"))),
                     torch.zeros(need, dtype=torch.uint8, device="cuda"))
    sampling, workspace = s["held"]
    fmx.call("fmx_sample", s["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"], ctypes.byref(sampling),
             s["uniform"].data_ptr(), s["ids"].data_ptr(), s["probs"].data_ptr(), workspace.data_ptr(),
             workspace.numel(), fmx.stream_handle())
    return {"ids": s["ids"], "probs": s["probs"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "attention": _own_attention, "sample": _own_sample}[kind](state)
    return {"rope": _plain_rope, "attention": _plain_attention, "sample": _plain_sample}[kind](state)


# -------------------------------------------------------------------- work --

def _pairs(case):
    """Visible (new token, position) pairs, and positions some token sees."""
    pairs = seen = 0
    window = case["window"] or 1 << 40
    for n, length in zip(*_counts(case)):
        first = length - n  # the first new token's position
        # token at p sees min(p + 1, window) positions
        whole = max(0, min(n, window - 1 - first))  # tokens that see all before them
        pairs += whole * first + whole * (whole + 1) // 2 + (n - whole) * window
        seen += length - max(0, first + 1 - window)
    return pairs, seen


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    H, kvh, D, size = case["heads"], case["kv_heads"], case["head_dim"], BYTES[case["type"]]
    tokens = sum(_counts(case)[0])
    if case["kind"] == "rope":
        elements = tokens * (H + 2 * kvh) * D
        return {"bytes": elements * (BYTES[case["source"]] + size), "flops": 3 * tokens * (H + kvh) * case["dims"]}
    pairs, seen = _pairs(case)
    return {"bytes": 2 * seen * kvh * D * size + tokens * H * D * (size + BYTES[case["out"]]),
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------- exact --

def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    H, kvh, D, R, ps = case["heads"], case["kv_heads"], case["head_dim"], case["dims"], case["page_size"]
    # complex numbers: a pair times magnitude e^(i angle)
    q_out, k, v = (s[n].double() for n in ("q_out", "k", "v"))
    starts, table = s["starts"].tolist(), s["table"].long()
    for i, (n, length) in enumerate(zip(*_counts(case))):
        position = torch.arange(length - n, length, device="cuda")
        x = s["qkv"][starts[i]:starts[i] + n].double().reshape(n, H + 2 * kvh, D).clone()
        turn = torch.polar(torch.full((n, R // 2), s["magnitude"], dtype=torch.float64, device="cuda"),
                           position.double()[:, None] * s["inv_freq"])
        part = x[:, :H + kvh, :R].clone()
        part = part.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (R // 2, 2))
        part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn[:, None, :])
        part = part.transpose(-1, -2) if case["layout"] == "half" else part
        x[:, :H + kvh, :R] = part.reshape(n, H + kvh, R)
        q_out[starts[i]:starts[i] + n] = x[:, :H]
        at = (table[i, position // ps], position % ps)
        _by_position(case, k)[at] = x[:, H:H + kvh]
        _by_position(case, v)[at] = x[:, H + kvh:]
    return {"q": q_out, "k": k, "v": v}


def _exact_attention(case, seed):
    s = _prepare_attention(case, seed)
    H, kvh, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    out = s["out"].double()
    starts, table = s["starts"].tolist(), s["table"].long()
    for i, (n, length) in enumerate(zip(*_counts(case))):
        j = torch.arange(length, device="cuda")
        page, place = table[i, j // ps], j % ps
        for h in range(kvh):
            k = _by_position(case, s["k"])[page, place, h].double()
            v = _by_position(case, s["v"])[page, place, h].double()
            step = max(1, (1 << 27) // length)
            for at in range(0, n, step):
                m = min(step, n - at)
                p = length - n + at + torch.arange(m, device="cuda")[:, None]
                hidden = j > p
                if case["window"]:
                    hidden |= j <= p - case["window"]
                for head in range(h * (H // kvh), (h + 1) * (H // kvh)):
                    row = slice(starts[i] + at, starts[i] + at + m)
                    a = (s["q"][row, head].double() / math.sqrt(D)) @ k.t()
                    if case["softcap"]:
                        a = case["softcap"] * torch.tanh(a / case["softcap"])
                    a[hidden] = -math.inf
                    if s["sinks"] is not None:
                        a = torch.cat((a, s["sinks"][head].double().expand(m, 1)), dim=1)
                    out[row, head] = torch.softmax(a, dim=1)[:, :length] @ v
    return out


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    R, V = case["rows"], case["vocab"]
    probs = torch.empty(R, dtype=torch.float64)
    for r in range(R):
        x = s["logits"][r].double()
        rank = torch.argsort(x, descending=True, stable=True)
        p = torch.softmax(x[rank] / s["temperature"][r].double(), dim=0)
        n = V if s["top_k"] is None else min(V, int(s["top_k"][r]))
        if s["top_p"] is not None:
            n = min(n, 1 + int((p[:n].cumsum(0) < s["top_p"][r].double() * p[:n].sum()).sum()))
        if s["min_p"] is not None:
            n = min(n, int((p >= s["min_p"][r].double() * p[0]).sum()))
        kept = p[:n] / p[:n].sum()
        probs[r] = kept[min(n - 1, int((kept.cumsum(0) <= s["uniform"][r].double()).sum()))]
    return {"ids": None, "probs": probs}


def exact(case, seed):
    return {"rope": _exact_rope, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](case, seed)
