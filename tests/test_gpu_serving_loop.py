"""The serving operators in the loop that uses them: a small decoder whose
projections, expert layer and head are libfmx's own, run with a prompt and then
token by token over pages, against the same decoder on fmx_attention_decode's
contiguous cache with rotary positions, sampling and prompt in plain torch."""
import ctypes
import math

import numpy as np
import pytest
import torch

import serving_ref as ref
from freemoe_amd import fmx
from freemoe_amd import serving as sv
from freemoe_amd import workloads as wl
from freemoe_amd.device import DeviceLayer, pack

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, VOCAB, LAYERS, PAGE = 256, 4, 2, 64, 500, 2, 8
WIDTH = (HEADS + 2 * KV) * DIM


class Decoder:
    def __init__(self, gpu):
        g = torch.Generator().manual_seed(77)
        self.gpu = gpu

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=g) / math.sqrt(cols)).to(gpu)

        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).to(gpu)
        self.qkv = [matrix(WIDTH, HIDDEN) for _ in range(LAYERS)]
        self.o = [matrix(HIDDEN, HEADS * DIM) for _ in range(LAYERS)]
        self.moe = [DeviceLayer(wl.make_layer(HIDDEN, 512, 4, 2, wl.Q8_0, 90 + i), gpu) for i in range(LAYERS)]
        self.head = matrix(VOCAB, HIDDEN) * 4
        self.rope = sv.Rope(DIM, layout=fmx.ROPE_HALF, device=gpu)

    def product(self, w, x):
        """y = x W^T row by row through fmx_gemm_quant, the batched product."""
        y = torch.empty(x.shape[0], w.shape[0], device=self.gpu)
        fmx.call("fmx_gemm_quant", fmx.FMX_TYPE_F32, w.data_ptr(), x.data_ptr(), y.data_ptr(), x.shape[0], w.shape[0],
                 w.shape[1], fmx.stream_handle())
        return y

    def norm(self, x):
        return x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5)


class Paged:
    """The decoder on the serving operators, several sequences at once."""

    def __init__(self, model, sequences, most):
        self.m, gpu = model, model.gpu
        pages = -(-most // PAGE)
        self.caches = [sv.Cache(sequences * pages, PAGE, KV, DIM, torch.float32, gpu) for _ in range(LAYERS)]
        order = torch.randperm(sequences * pages, generator=torch.Generator().manual_seed(3))
        self.table = order.to(torch.int32).reshape(sequences, pages).to(gpu)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=gpu)

    def step(self, ids, counts):
        """Logits of each sequence's last new token; ids: all new tokens in order."""
        m, gpu, T = self.m, self.m.gpu, sum(counts)
        starts = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=gpu)
        self.lengths += torch.tensor(counts, dtype=torch.int32, device=gpu)
        batch = sv.Batch(starts, self.lengths, self.table, T, max(counts))
        x = m.embed[ids]
        for layer in range(LAYERS):
            qkv = m.product(m.qkv[layer], m.norm(x)).reshape(T, HEADS + 2 * KV, DIM)
            q = torch.empty(T, HEADS, DIM, device=gpu)
            ws = sv.attention_workspace(self.caches[layer], batch, HEADS)
            sv.rope_append(self.caches[layer], batch, m.rope, qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:], q, ws)
            a = torch.empty(T, HEADS, DIM, device=gpu)
            sv.attention(self.caches[layer], batch, q, a, ws)
            assert sv.status(ws) == 0
            x = x + m.product(m.o[layer], a.reshape(T, -1))
            x, _, _ = m.moe[layer].decode(x.contiguous())
        last = (starts[1:] - 1).long()
        return m.product(m.head, m.norm(x[last]))


class Plain:
    """One sequence, one token at a time, on fmx_attention_decode and torch."""

    def __init__(self, model, most):
        self.m = model
        self.kv = [torch.zeros(most, 2 * KV * DIM, device=model.gpu) for _ in range(LAYERS)]
        self.n = 0

    def token(self, i):
        m, gpu = self.m, self.m.gpu
        x = m.embed[i:i + 1]
        for layer in range(LAYERS):
            qkv = m.product(m.qkv[layer], m.norm(x)).reshape(1, HEADS + 2 * KV, DIM)
            turned, _ = ref.rope(qkv.cpu()[:, :HEADS + KV], torch.tensor([self.n]), m.rope.inv_freq.cpu(), 1.0, DIM, True)
            turned = turned.float().to(gpu)
            self.kv[layer][self.n] = torch.cat((turned[0, HEADS:].reshape(-1), qkv[0, HEADS + KV:].reshape(-1)))
            q, a = turned[0, :HEADS].reshape(-1).contiguous(), torch.empty(HEADS * DIM, device=gpu)
            ws = torch.zeros(256, dtype=torch.uint8, device=gpu)
            fmx.call("fmx_attention_decode", q.data_ptr(), self.kv[layer].data_ptr(), 2 * KV * DIM, KV * DIM, HEADS, KV,
                     DIM, self.n + 1, 1.0 / math.sqrt(DIM), a.data_ptr(), ws.data_ptr(), 256, fmx.stream_handle())
            x = x + m.product(m.o[layer], a.reshape(1, -1))
            x, _, _ = m.moe[layer].decode(x.contiguous())
        self.n += 1
        return m.product(m.head, m.norm(x))


def test_prompt_and_tokens_over_pages(gpu):
    m = Decoder(gpu)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (37, 1, 90)]
    steps, most = 12, 110
    paged = Paged(m, len(prompts), most)
    plain = [Plain(m, most) for _ in prompts]
    logits = paged.step(torch.tensor(sum(prompts, []), device=gpu), [len(p) for p in prompts])
    want = []
    for p, prompt in zip(plain, prompts):
        for i in prompt:
            last = p.token(i)
        want.append(last)
    settings = dict(temperature=torch.full((3,), 0.8, device=gpu), top_k=torch.full((3,), 40, dtype=torch.int32, device=gpu),
                    top_p=torch.full((3,), 0.9, device=gpu))
    for _ in range(steps):
        want = torch.cat(want)
        # two decoders that round differently in rotary positions, attention (f32
        # sums against double ones) and nowhere else: some 2^-20 of a logit's size
        # after 2 layers, and 16 times that allowed
        assert (logits - want).abs().max() <= 2.0 ** -16 * want.abs().max()
        u = torch.rand(3, generator=g)
        ids, probs = sv.sample(logits, u.to(gpu), **settings)
        for r in range(3):
            i, p = ref.sample(logits[r].cpu(), float(u[r]), temperature=float(np.float32(0.8)), top_k=40, top_p=float(np.float32(0.9)))
            assert int(ids[r]) == i and abs(float(probs[r]) - p) <= 1e-6
        logits = paged.step(ids.long(), [1, 1, 1])
        want = [p.token(int(i)) for p, i in zip(plain, ids.tolist())]
