"""GPU: a decoder block served by the operators together: page tables, norms with 8-bit
output, adapters, rotary positions, the paged cache and attention; against the block in fp32, in
any split of the tokens into steps, and replayed from a graph."""
import importlib.util
import os

import pytest
import torch

from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "quantized_block.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("quantized_block", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits,tokens,steps,limit", [(8, 200, 8, 0.05), (8, 3, 3, 0.05),
                                                     (4, 150, 4, 0.15)])
def test_block_follows_its_fp32_form(dev, example, bits, tokens, steps, limit):
    """A group of 8 bits has noise of about range/255/√12, under 1 % of its values'
    size for normal data, in each of some ten roundings; an output is the sum of the input,
    which has none, and of two branches of about its size: 5 % in all is ample.  With 4 bits,
    keys' and values' noise is about 12 % of their size each, in one of the branches."""
    outs, refs = example.serve(bits=bits, tokens=tokens, steps=steps, device="cuda:0")
    for y, ref in zip(outs, refs):
        assert y.shape == ref.shape and y.dtype is torch.bfloat16
        assert bool(torch.isfinite(y).all())
        err = float((y.float() - ref).norm() / ref.norm())
        print(f"{bits} bits, {len(y)} tokens: relative error {err:.4f}")
        assert err < limit


def _block(example, dev, pages=60, requests=6):
    return example.Block(example.weights(gen(1), dev), pages, requests, 160, 8)


@torch.no_grad()
def test_replayed_steps_are_the_eager_ones(dev, example):
    """Single tokens from a graph, each replay with the next token's pages, beside the same
    steps of another block without a graph; other eager work in between."""
    i32 = dict(dtype=torch.int32, device=dev)
    rows, index = torch.tensor([5, 1, 3], **i32), torch.tensor([0, -1, 1], **i32)
    new, one = torch.tensor([17, 1, 30], **i32), torch.ones(3, **i32)
    blocks = [_block(example, dev) for _ in range(2)]
    g = gen(2)
    prompt = torch.randn(48, example.HIDDEN, generator=g).bfloat16().to(dev)
    for b in blocks:
        b(prompt, rows, new, index.repeat_interleave(new.long()))
    tokens = torch.randn(40, 3, example.HIDDEN, generator=g).bfloat16().to(dev)
    x = tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a step ahead of the capture, then undone
        blocks[0](x, rows, one, index)
        blocks[0].tables.release(rows, new)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = blocks[0](x, rows, one, index)
    for i in range(40):
        x.copy_(tokens[i])
        graph.replay()
        want = blocks[1](tokens[i], rows, one, index)
        torch.cuda.synchronize()
        assert_bitexact(y, want, f"step {i}")
    for b in blocks:
        b.check()
    assert_bitexact(blocks[0].tables.table, blocks[1].tables.table, "tables")


@torch.no_grad()
def test_a_request_does_not_depend_on_its_batch(dev, example):
    """The same request's single tokens beside others, in another place of the batch, and with a
    draft taken back in between: the same bits, and the same pages afterwards."""
    i32 = dict(dtype=torch.int32, device=dev)
    a, b = (_block(example, dev) for _ in range(2))
    g = gen(3)
    mine = torch.randn(20, example.HIDDEN, generator=g).bfloat16().to(dev)
    other = torch.randn(20, example.HIDDEN, generator=g).bfloat16().to(dev)
    row, both = torch.tensor([2], **i32), torch.tensor([4, 2], **i32)
    one = torch.ones(2, **i32)
    for i in range(20):
        alone = a(mine[i:i + 1], row, one[:1], one[:1])
        held = b.tables.lengths[both.long()].clone()
        b(other[:6], both, torch.tensor([2, 4], **i32), torch.zeros(6, **i32))
        b.tables.release(both, held)
        beside = b(torch.stack([other[i], mine[i]]), both, one, one)
        assert_bitexact(beside[1:], alone, f"token {i}")
    a.check()
    b.check()


@torch.no_grad()
def test_two_streams_at_once(dev, example):
    """Two blocks served on a stream each: no workspace is shared."""
    i32 = dict(dtype=torch.int32, device=dev)
    rows, index = torch.tensor([5, 1], **i32), torch.tensor([0, 1], **i32)
    g = gen(4)
    steps = [[torch.randn(n, example.HIDDEN, generator=g).bfloat16().to(dev) for n in (130, 2, 2, 2)]
             for _ in range(2)]
    counts = [torch.tensor(n, **i32) for n in ([100, 30], [1, 1], [1, 1], [1, 1])]

    def serve(block, xs):
        return [block(x, rows, n, index.repeat_interleave(n.long(), output_size=len(x)))
                for x, n in zip(xs, counts)]

    want = [serve(_block(example, dev), xs) for xs in steps]
    blocks = [_block(example, dev) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(4):
        for b in range(2):
            with torch.cuda.stream(streams[b]):
                n = counts[i]
                got[b].append(blocks[b](steps[b][i], rows, n, index.repeat_interleave(
                    n.long(), output_size=len(steps[b][i]))))
    torch.cuda.synchronize()
    for b in range(2):
        for i, (y, ref) in enumerate(zip(got[b], want[b])):
            assert_bitexact(y, ref, f"stream {b} step {i}")
