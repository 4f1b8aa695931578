"""A self-attention layer run on what its quantization made: 8-bit linears from
GPTQ's exported codes, a quantized paged cache, and attention over it.

    python examples/quantized_layer.py [--bits 4|8] [--tokens N] [--steps N]

Calibrates and quantizes the four projections (8 bits, one scale per output
channel), exports them, and serves two sequences of different lengths: their
prompts in two chunks each, then single tokens.  Prints how far the outputs
are from the same layer in fp32.
"""
import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from g2ptq_amd import (GPTQ, Int8Linear, PagedKVCache, WeightQuantizer,  # noqa: E402
                       make_group_quantizers, paged_attention)

HIDDEN, HEADS, KV_HEADS, DIM, PAGE = 1024, 8, 2, 128, 16


def projections(generator, device):
    """The layer's q, k, v and output projections."""
    def linear(rows, cols):
        lin = torch.nn.Linear(cols, rows, bias=False)
        with torch.no_grad():
            lin.weight.copy_(torch.randn(rows, cols, generator=generator) / math.sqrt(cols))
        return lin.to(device)
    return {"q": linear(HEADS * DIM, HIDDEN), "k": linear(KV_HEADS * DIM, HIDDEN),
            "v": linear(KV_HEADS * DIM, HIDDEN), "o": linear(HIDDEN, HEADS * DIM)}


def quantize(linear, calibration):
    """GPTQ at 8 bits per channel, exported, as a linear that runs in 8-bit integers."""
    layer = torch.nn.Linear(linear.in_features, linear.out_features, bias=False,
                            device=linear.weight.device)
    layer.weight.data.copy_(linear.weight.data)
    gptq = GPTQ([layer])
    quantizer = WeightQuantizer()
    quantizer.configure(8, perchannel=True, sym=True)
    gptq.quantizer = make_group_quantizers(quantizer, linear.in_features, -1)
    gptq.add_batch(0, calibration.unsqueeze(0), None)
    gptq.fasterquant(blocksize=128, percdamp=0.01, groupsize=-1, backend="hip",
                     export_compressed_tensors=True)
    gptq.free()
    return Int8Linear.from_export(layer)


class Layer:
    """The quantized layer and its cache."""

    def __init__(self, linears, calibration, pages, bits):
        dev = calibration.device
        with torch.no_grad():
            attended = calibration @ linears["v"].weight.t()  # the size of the output's inputs
            attended = attended.repeat(1, HEADS // KV_HEADS)
        inputs = {"q": calibration, "k": calibration, "v": calibration, "o": attended}
        self.lin = {name: quantize(linears[name], inputs[name]) for name in linears}
        self.cache = PagedKVCache(pages, PAGE, KV_HEADS, DIM, bits=bits, sym=bits == 8, device=dev)

    def __call__(self, x, table, cu, lengths, slots):
        """``x`` (tokens, HIDDEN): each sequence's next tokens, whose cache slots are
        ``slots``; ``lengths`` counts them in."""
        n = x.shape[0]
        q = self.lin["q"](x).view(n, HEADS, DIM)
        k = self.lin["k"](x).view(n, KV_HEADS, DIM)
        v = self.lin["v"](x).view(n, KV_HEADS, DIM)
        self.cache.write(k, v, slots)
        out = paged_attention(q, self.cache, table, cu, lengths)
        return self.lin["o"](out.view(n, HEADS * DIM))


def reference(linears, x):
    """The same layer in fp32 on one whole sequence."""
    n = x.shape[0]
    x = x.float()
    q, k, v = (linears[m](x).view(n, -1, DIM).transpose(0, 1) for m in "qkv")
    k, v = (t.repeat_interleave(HEADS // KV_HEADS, dim=0) for t in (k, v))
    logits = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(DIM)
    mask = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
    p = logits.masked_fill(mask, -math.inf).softmax(-1)
    return linears["o"](torch.bmm(p, v.contiguous()).transpose(0, 1).reshape(n, HEADS * DIM))


@torch.no_grad()
def serve(bits=8, tokens=200, steps=8, device="cuda", seed=0):
    """Runs two sequences through the layer in chunks and single tokens; returns
    each one's outputs and the fp32 reference's."""
    g = torch.Generator().manual_seed(seed)
    linears = projections(g, device)
    calibration = torch.randn(2048, HIDDEN, generator=g).to(device)
    prompts = [tokens, max(2, tokens // 3)]
    xs = [torch.randn(p + steps, HIDDEN, generator=g).to(device).bfloat16() for p in prompts]
    need = [-(-len(x) // PAGE) for x in xs]
    layer = Layer(linears, calibration, sum(need), bits)
    # pages are dealt out in turn, so that neither sequence's are consecutive
    table = torch.zeros(2, max(need), dtype=torch.int32)
    deal = [(i, b) for i in range(max(need)) for b in range(2) if i < need[b]]
    for page, (i, b) in enumerate(deal):
        table[b, i] = page
    outs, done = [[], []], [0, 0]
    halves = [p // 2 for p in prompts]
    rounds = [halves, [p - h for p, h in zip(prompts, halves)]] + [[1, 1]] * steps
    on_device = table.to(device)
    for news in rounds:
        x = torch.cat([xs[b][done[b]:done[b] + n] for b, n in enumerate(news)])
        slots = torch.tensor([int(table[b, p // PAGE]) * PAGE + p % PAGE
                              for b, n in enumerate(news) for p in range(done[b], done[b] + n)])
        done = [d + n for d, n in zip(done, news)]
        y = layer(x, on_device, torch.tensor([0, news[0], sum(news)], dtype=torch.int32,
                                             device=device),
                  torch.tensor(done, dtype=torch.int32, device=device), slots.to(device))
        for b, part in enumerate(y.split(list(news))):
            outs[b].append(part)
    layer.cache.check()
    return [torch.cat(o) for o in outs], [reference(linears, x) for x in xs]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--bits", type=int, choices=(4, 8), default=8)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    outs, refs = serve(a.bits, a.tokens, a.steps)
    for b, (y, ref) in enumerate(zip(outs, refs)):
        err = float((y.float() - ref).norm() / ref.norm())
        print(f"sequence {b}: {len(y)} tokens, relative error {err:.4f} "
              f"(8-bit linears, {a.bits}-bit cache)")


if __name__ == "__main__":
    main()
