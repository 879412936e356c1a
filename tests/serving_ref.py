"""Plain statements of the serving operators in 64 bits, on the host: rotary
positions with the cache write, attention over pages, sampling."""
import math

import torch


class Paged:
    """A ragged batch with its pools, made on the host: sequence i has lengths[i]
    positions, the last counts[i] of them new. Every pool value that no position
    owns, and every table entry behind a sequence's pages, is poison."""

    def __init__(self, counts, lengths, kv_heads, head_dim, page_size, dtype, seed, by_head=False, spare=2,
                 pad=0, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.counts, self.lengths, self.page_size = counts, lengths, page_size
        need = [-(-n // page_size) for n in lengths]
        pages = max(1, sum(need) + 2)
        order = torch.randperm(pages, generator=g).tolist()
        stride = max(need + [1]) + 1
        self.table = torch.full((len(counts), stride), -1, dtype=torch.int32)
        self.pages = []
        for i, n in enumerate(need):
            mine, order = order[:n], order[n:]
            self.table[i, :n] = torch.tensor(mine, dtype=torch.int32)
            self.pages.append(mine)
        shape = (pages, kv_heads, page_size, head_dim + pad) if by_head else (pages, page_size, kv_heads, head_dim + pad)
        self.pools = []
        for _ in range(2):
            pool = torch.full(shape, float("nan"), dtype=dtype)
            view = pool[..., :head_dim].transpose(1, 2) if by_head else pool[..., :head_dim]
            for mine, n in zip(self.pages, lengths):
                for j, page in enumerate(mine):
                    m = min(page_size, n - j * page_size)
                    view[page, :m] = (torch.randn(m, kv_heads, head_dim, generator=g) * scale).to(dtype)
            self.pools.append((pool, view))
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.tokens, self.max_new = self.starts[-1] + spare, max(counts + [1])
        self.by_head, self.head_dim, self.g = by_head, head_dim, g

    def rows(self, i, which):
        """Sequence i's positions of a pool, [length, kv heads, head_dim] (a copy)."""
        view = self.pools[which][1]
        j = torch.arange(self.lengths[i])
        return view[self.table[i].long()[j // self.page_size], j % self.page_size]

    def on(self, device):
        """The serving module's Cache and Batch on the device."""
        from freemoe_amd import serving as sv
        pools = [p.to(device) for p, _ in self.pools]
        views = [p[..., :self.head_dim].transpose(1, 2) if self.by_head else p[..., :self.head_dim] for p in pools]
        cache = sv.Cache.of(*views)
        batch = sv.Batch(torch.tensor(self.starts, dtype=torch.int32).to(device),
                         torch.tensor(self.lengths, dtype=torch.int32).to(device), self.table.to(device), self.tokens,
                         self.max_new)
        return cache, batch


def attention(paged, q, scale, softcap=0.0, window=0, sinks=None):
    """Per sequence (row slice, out, spread) in float64: spread is sum_j p_j |v_j|,
    what a relative error of the weights moves an output by; and the largest
    sum_d |q_d k_jd| scale of each row and head."""
    heads = q.shape[1]
    for i, (n, length) in enumerate(zip(paged.counts, paged.lengths)):
        k, v = paged.rows(i, 0).double(), paged.rows(i, 1).double()
        kvh = k.shape[1]
        rows = slice(paged.starts[i], paged.starts[i] + n)
        out, spread = torch.zeros(n, heads, q.shape[2], dtype=torch.float64), torch.zeros(n, heads, q.shape[2], dtype=torch.float64)
        size = torch.zeros(n, heads, 1, dtype=torch.float64)
        for r in range(n):
            p = length - n + r
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                continue
            for h in range(heads):
                kk, vv = k[lo:p + 1, h // (heads // kvh)], v[lo:p + 1, h // (heads // kvh)]
                qq = q[paged.starts[i] + r, h].double()
                s = kk @ qq * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                top = s.max() if sinks is None else torch.maximum(s.max(), sinks[h].double())
                w = torch.exp(s - top)
                w = w / (w.sum() + (0.0 if sinks is None else torch.exp(sinks[h].double() - top)))
                out[r, h] = w @ vv
                spread[r, h] = w @ vv.abs()
                size[r, h] = (kk.abs() @ qq.abs()).max() * abs(scale)
        yield rows, out, spread, size


def rope(x, positions, inv_freq, magnitude, dims, half):
    """x [tokens, heads, head_dim] turned at its positions, float64; and a bound's
    size: |x| + |y| of each element's pair times the magnitude (0 where copied)."""
    x = x.double()
    angle = positions.double()[:, None] * inv_freq
    cos, sin = torch.cos(angle)[:, None] * magnitude, torch.sin(angle)[:, None] * magnitude
    c = torch.arange(dims // 2)
    a, b = (c, c + dims // 2) if half else (2 * c, 2 * c + 1)
    out, size = x.clone(), torch.zeros_like(x)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., a] * sin + x[..., b] * cos
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(magnitude)
    return out, size


def sample(x, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, probability) for one row, float64 (temperature and the rest as Python
    floats that hold their float32 values)."""
    x = x.double()
    x = torch.where(x == 0, 0.0, x)  # -0 and 0 are equal
    order = torch.argsort(x, descending=True, stable=True)
    if temperature == 0.0:
        return int(order[0]), 1.0
    # (-inf carries no weight, at an infinite temperature either, where -inf / inf is NaN)
    w = torch.where(x[order] == -math.inf, 0.0, torch.exp((x[order] - x[order[0]]) / temperature))
    n = len(w) if top_k == 0 else min(top_k, len(w))
    mass = torch.cumsum(w, 0)
    if top_p < 1.0:
        n = min(n, 1 + int((mass[:n] < top_p * mass[n - 1]).sum()))
    if min_p > 0.0:
        n = max(1, min(n, int((w >= min_p).sum())))
    at = min(n - 1, int((mass[:n] <= min(uniform, 1.0 - 2.0 ** -24) * mass[n - 1]).sum()))
    return int(order[at]), float(w[at] / mass[n - 1])


def bound_of(dtype):
    """Half a step of a type's normal values, relative."""
    return torch.finfo(dtype).eps / 2


def half_step(dtype, value):
    """Half a step of a type at `value`: relative, and below the smallest normal
    value (2^-14 for a half, whose steps there are 2^-24) that of the steps there,
    smallest_normal x eps."""
    info = torch.finfo(dtype)
    return torch.clamp_min(value.abs() * info.eps / 2, info.smallest_normal * info.eps / 2)
