"""A decoder block served in 8-bit integers: page tables, norms that give 8-bit codes, low-rank
adapters of each request, rotary positions, a quantized paged cache and attention over it.

    python examples/quantized_block.py [--bits 4|8] [--tokens N] [--steps N]

Serves three requests of different lengths, each with its own adapter or none: their prompts in
two chunks each, then single tokens, in batches whose tokens are padded.  Prints how far the
outputs are from the same block in fp32.
"""
import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from g2ptq_amd import (Int8Linear, LowRankAdapters, PagedKVCache, PageTables, Rotary,  # noqa: E402
                       WeightQuantizer, int8_matmul, paged_attention, rms_norm, rms_norm_quantize)

HIDDEN, HEADS, KV_HEADS, DIM, INNER, PAGE, EPS = 1024, 8, 2, 128, 2048, 16, 1e-5
SIZES = {"q": (HEADS * DIM, HIDDEN), "k": (KV_HEADS * DIM, HIDDEN), "v": (KV_HEADS * DIM, HIDDEN),
         "o": (HIDDEN, HEADS * DIM), "gate": (INNER, HIDDEN), "up": (INNER, HIDDEN),
         "down": (HIDDEN, INNER)}
ADAPTED, RANKS, SCALE = ("q", "v", "down"), (16, 8), 0.5


def weights(generator, device):
    """The block's linears, norms and adapters, in fp32."""
    def randn(*shape):
        return torch.randn(*shape, generator=generator).to(device)
    w = {name: randn(*size) / math.sqrt(size[1]) for name, size in SIZES.items()}
    w |= {name: 1 + 0.2 * randn(n) for name, n in (("norm", HIDDEN), ("norm2", HIDDEN),
                                                   ("q_norm", DIM), ("k_norm", DIM))}
    w |= {name + "_down": [(randn(r, SIZES[name][1]) / math.sqrt(SIZES[name][1])).bfloat16()
                           for r in RANKS] for name in ADAPTED}
    w |= {name + "_up": [(randn(SIZES[name][0], r) / math.sqrt(r)).bfloat16() for r in RANKS]
          for name in ADAPTED}
    return w


def quantized(weight):
    linear = torch.nn.Linear(weight.shape[1], weight.shape[0], bias=False, device=weight.device)
    linear.weight.data.copy_(weight)
    quantizer = WeightQuantizer()
    quantizer.configure(8, perchannel=True, sym=True)
    quantizer.find_params(linear.weight.data)
    return Int8Linear.from_linear(linear, quantizer)


class Block:
    """The block, its cache and its requests' pages."""

    def __init__(self, w, pages, requests, length, bits):
        dev = w["norm"].device
        self.w = w
        self.lin = {name: quantized(w[name]) for name in SIZES}
        self.adapters = {name: LowRankAdapters(w[name + "_down"], w[name + "_up"], scale=SCALE)
                         for name in ADAPTED}
        self.rotary = Rotary(DIM, base=500000.0, device=dev)
        self.cache = PagedKVCache(pages, PAGE, KV_HEADS, DIM, bits=bits, sym=bits == 8, device=dev)
        self.tables = PageTables(pages, PAGE, requests, -(-length // PAGE), device=dev)

    def project(self, name, t, index):
        """A projection of normed tokens and, where it has adapters, each token's own."""
        y = int8_matmul(t.codes, t.scale, self.lin[name])
        return self.adapters[name].add_(y, t.values, index) if name in self.adapters else y

    def __call__(self, x, rows, new, index):
        """``x`` (tokens, HIDDEN): the next ``new[i]`` tokens of the requests in ``rows``, then
        padding; ``index``: every token's adapter."""
        n, w = x.shape[0], self.w
        step = self.tables.extend(rows, new, n)
        t = rms_norm_quantize(x, w["norm"], EPS, values=True)
        q = rms_norm(self.project("q", t, index).view(n, HEADS, DIM), w["q_norm"], EPS)
        k = rms_norm(self.project("k", t, index).view(n, KV_HEADS, DIM), w["k_norm"], EPS)
        v = self.project("v", t, index).view(n, KV_HEADS, DIM)
        q, k = self.rotary(q, k, step.positions)
        self.cache.write(k, v, step.slots)
        a = paged_attention(q, self.cache, step.table, step.cu, step.kv_lens)
        t = rms_norm_quantize(self.lin["o"](a.view(n, HEADS * DIM)), w["norm2"], EPS, residual=x,
                              values=True)
        inner = torch.nn.functional.silu(self.project("gate", t, index))
        inner *= self.project("up", t, index)
        return t.sum + self.adapters["down"](inner, index, base=self.lin["down"](inner))

    def check(self):
        self.tables.check()
        self.cache.check()
        for a in self.adapters.values():
            a.check()


def reference(w, x, adapter):
    """The same block in fp32 on one whole sequence."""
    def norm(x, weight):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight

    def project(name, x):
        y = x @ w[name].t()
        if name in ADAPTED and adapter >= 0:
            y = y + SCALE * (x @ w[name + "_down"][adapter].float().t()
                             @ w[name + "_up"][adapter].float().t())
        return y

    def turn(x):
        theta = 500000.0 ** (-torch.arange(0, DIM, 2, device=x.device, dtype=torch.float64) / DIM)
        angle = torch.arange(len(x), device=x.device).double()[:, None] * theta
        c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    n, x = len(x), x.float()
    h = norm(x, w["norm"])
    q = turn(norm(project("q", h).view(n, HEADS, DIM), w["q_norm"])).transpose(0, 1)
    k = turn(norm(project("k", h).view(n, KV_HEADS, DIM), w["k_norm"])).transpose(0, 1)
    v = project("v", h).view(n, KV_HEADS, DIM).transpose(0, 1)
    k, v = (t.repeat_interleave(HEADS // KV_HEADS, dim=0) for t in (k, v))
    logits = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(DIM)
    mask = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
    p = logits.masked_fill(mask, -math.inf).softmax(-1)
    x = x + project("o", torch.bmm(p, v.contiguous()).transpose(0, 1).reshape(n, HEADS * DIM))
    h = norm(x, w["norm2"])
    return x + project("down", torch.nn.functional.silu(project("gate", h)) * project("up", h))


@torch.no_grad()
def serve(bits=8, tokens=200, steps=8, device="cuda", seed=0, padding=3):
    """Runs three requests through the block in chunks and single tokens; returns each one's
    outputs and the fp32 reference's."""
    g = torch.Generator().manual_seed(seed)
    w = weights(g, device)
    prompts, adapters = [tokens, max(2, tokens // 3), max(2, tokens // 7)], [1, -1, 0]
    xs = [torch.randn(p + steps, HIDDEN, generator=g).to(device).bfloat16() for p in prompts]
    longest = max(len(x) for x in xs)
    pages = sum(-(-len(x) // PAGE) for x in xs)
    block = Block(w, pages, 5, longest, bits)
    i32 = dict(dtype=torch.int32, device=device)
    rows = torch.tensor([4, 0, 2], **i32)
    outs, done = [[] for _ in xs], [0] * len(xs)
    halves = [p // 2 for p in prompts]
    rounds = [halves, [p - h for p, h in zip(prompts, halves)]] + [[1] * len(xs)] * steps
    for news in rounds:
        part = [x[d:d + n] for x, d, n in zip(xs, done, news)]
        done = [d + n for d, n in zip(done, news)]
        pad = torch.zeros(padding, HIDDEN, dtype=torch.bfloat16, device=device)
        index = [a for a, n in zip(adapters, news) for _ in range(n)] + [-1] * padding
        y = block(torch.cat(part + [pad]), rows, torch.tensor(news, **i32),
                  torch.tensor(index, **i32))
        for out, piece in zip(outs, y.split(list(news) + [padding])):
            out.append(piece)
    block.check()
    block.tables.release(rows)
    assert int(block.tables.free_count) == pages
    return [torch.cat(o) for o in outs], [reference(w, x, a) for x, a in zip(xs, adapters)]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--bits", type=int, choices=(4, 8), default=8)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    outs, refs = serve(a.bits, a.tokens, a.steps)
    for b, (y, ref) in enumerate(zip(outs, refs)):
        err = float((y.float() - ref).norm() / ref.norm())
        print(f"request {b}: {len(y)} tokens, relative error {err:.4f} "
              f"(8-bit linears, {a.bits}-bit cache)")


if __name__ == "__main__":
    main()
