"""GPU: attention over the paged cache against fp64 on the values the cache holds,
within a bound derived from the roundings the kernels make: ragged chunks and
single tokens, shared heads, head sizes, bits and grids, pages that end inside a
tile, queries without keys, bad values in keys a query does not see."""
import pytest
import torch

from oracle import serving
from tests._util import assert_bitexact, gen
from tests.test_gpu_kv_cache import make_batch, offsets, values

pytestmark = pytest.mark.gpu


class Batch:
    def __init__(self, dev, q_lens, kv_lens, heads, kv_heads, dim, page, bits, sym, dtype,
                 seed=1, edit=None):
        from g2ptq_amd import PagedKVCache
        self.q_lens, self.kv_lens = q_lens, kv_lens
        self.table, pool = make_batch(seed, kv_lens, page)
        self.cache = PagedKVCache(pool, page, kv_heads, dim, bits=bits, sym=sym, device=dev)
        cu = offsets(kv_lens).tolist()
        k, v = (values(cu[-1], kv_heads, dim, dtype, seed + s) for s in (1, 2))
        q = values(sum(q_lens), heads, dim, dtype, seed + 3)
        if edit:
            edit(q, k, v, cu)
        self.q, self.dim, self.dev, self.dtype = q.to(dev), dim, dev, dtype
        self.cache.write(k.to(dev), v.to(dev),
                         serving.slot_map(self.table, page, cu, kv_lens).to(dev))
        self.k, self.v = ([serving.dequantize(*serving.quantize(x, bits, sym))[a:b]
                           for a, b in zip(cu, cu[1:])] for x in (k, v))
        span = serving.quantize(v, bits, sym)[1].double() * (2 ** bits - 1)
        self.span = [span[a:b] for a, b in zip(cu, cu[1:])]

    def run(self, q=None, **kw):
        from g2ptq_amd import paged_attention
        return paged_attention(self.q if q is None else q, self.cache, self.table.to(self.dev),
                               offsets(self.q_lens).to(self.dev),
                               torch.tensor(self.kv_lens, dtype=torch.int32, device=self.dev),
                               **kw)

    def check(self, out, what="", scale=None, rows=None):
        scale = serving.default_scale(self.dim) if scale is None else scale
        ref, size, logit, span, count = serving.attention(
            self.q.cpu(), self.k, self.v, offsets(self.q_lens).tolist(), self.kv_lens, scale,
            self.span)
        bound = serving.attention_bound(self.dtype, ref, size, logit, span, count, self.dim)
        assert out.dtype is self.dtype and out.shape == ref.shape
        err = (out.cpu().double() - ref).abs()
        ok = err <= bound
        if rows is not None:
            ok = ok[rows]
        assert bool(ok.all()), (what, float((err / bound)[~bound.isnan()].max()))
        empty = count == 0
        assert bool((out.cpu()[empty] == 0).all()), what
        self.cache.check()
        return ref


CHUNKS = [
    ([1], [1]), ([1], [37]), ([1], [700]), ([5], [5]), ([33], [40]), ([70], [70]),
    ([130], [300]), ([1, 1, 1, 1], [1, 64, 65, 200]), ([3, 0, 1, 20, 64], [3, 9, 0, 20, 129]),
    ([2, 17, 1], [1, 5, 0]),  # queries without keys
    ([16, 16], [1000, 31]), ([257], [257]),
]


@pytest.mark.parametrize("bits,sym", [(8, True), (8, False), (4, True), (4, False)])
@pytest.mark.parametrize("q_lens,kv_lens", CHUNKS, ids=str)
def test_ragged_chunks(dev, q_lens, kv_lens, bits, sym):
    for dtype, heads, kv_heads, dim, page in ((torch.bfloat16, 8, 2, 128, 16),
                                              (torch.float16, 3, 1, 64, 64)):
        b = Batch(dev, q_lens, kv_lens, heads, kv_heads, dim, page, bits, sym, dtype)
        b.check(b.run(), f"{dtype}")
        b.check(b.run(max_q=max(q_lens), max_kv=max(kv_lens)), f"{dtype} sized")


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [
    (1, 1, 16, 1), (4, 4, 32, 2), (6, 2, 48, 8), (5, 1, 80, 16), (16, 1, 96, 32), (32, 2, 112, 64),
    (7, 7, 128, 128), (40, 1, 64, 256), (4, 2, 160, 16), (8, 4, 192, 4096), (2, 1, 240, 16),
    (12, 3, 256, 32), (128, 1, 128, 16)])
def test_heads_dims_and_pages(dev, heads, kv_heads, dim, page, bits):
    for q_lens, kv_lens in (([1, 1], [90, 33]), ([9, 70, 1], [9, 75, 150])):
        b = Batch(dev, q_lens, kv_lens, heads, kv_heads, dim, page, bits, False, torch.bfloat16,
                  seed=dim)
        b.check(b.run(), f"{q_lens}")


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [9001]), ([1, 1, 1], [5000, 1, 2500]),
                                            ([4], [6000]), ([40, 1], [3100, 4200])], ids=str)
@pytest.mark.parametrize("bits", [8, 4])
def test_long_contexts_with_few_rows(dev, q_lens, kv_lens, bits):
    b = Batch(dev, q_lens, kv_lens, 8, 2, 128, 64, bits, True, torch.float16)
    b.check(b.run())
    # sizes given far too small only shape the launch
    b.check(b.run(max_q=1, max_kv=1), "small hints")
    b.check(b.run(max_q=0, max_kv=0), "no hints")


@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads,dim", [
    ([300, 20, 100], [4000, 20, 900], 4, 2, 64),       # chunks in as many shares as they need
    ([90, 1, 2, 40], [1500, 3000, 20, 41], 4, 2, 48),  # and short ones with them
    ([1] * 64, [5200] + [(37 * i) % 900 for i in range(1, 64)], 8, 8, 16),
    ([2] * 20, [1 + (613 * i) % 3000 for i in range(20)], 2, 1, 32)],
    ids=["chunks", "mixed", "many", "pairs"])
def test_batches_of_sequences_of_very_different_lengths(dev, q_lens, kv_lens, heads, kv_heads,
                                                        dim):
    b = Batch(dev, q_lens, kv_lens, heads, kv_heads, dim, 16, 8, False, torch.bfloat16)
    b.check(b.run(max_q=max(q_lens), max_kv=max(kv_lens)), "sized")
    b.check(b.run(max_q=max(q_lens), max_kv=300), "lengths beyond the stated one")
    b.check(b.run(max_q=1, max_kv=max(kv_lens)), "more rows than stated")
    b.check(b.run(), "unsized")


def test_scale_and_strides(dev):
    b = Batch(dev, [20, 1], [50, 77], 4, 2, 64, 16, 8, False, torch.bfloat16)
    for scale in (0.0, -0.3, 1.0):
        b.check(b.run(scale=scale), f"scale {scale}", scale=scale)
    base = b.run()
    wide = torch.zeros(21, 9, 67, dtype=torch.bfloat16, device=dev)
    wide[:, 2:6, 3:] = b.q
    assert_bitexact(b.run(q=wide[:, 2:6, 3:]), base, "offset view")
    apart = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert_bitexact(b.run(q=apart), base, "heads first")
    last = b.q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert_bitexact(b.run(q=last), base, "channels first")


@pytest.mark.parametrize("q_lens,kv_lens", [([40], [60]), ([200], [210]), ([1], [60])], ids=str)
def test_large_and_small_values(dev, q_lens, kv_lens):
    """Queries and keys over the types' ranges, values whose sizes differ by 2^20
    between tokens, logits far apart (a softmax on one key)."""
    def edit(q, k, v, cu):
        q[0] *= 1e-4
        q[-1] = (q[-1].float() * 30).to(q.dtype)
        v[::3] = (v[::3].float() * 2.0 ** -10).to(v.dtype)
        v[1::7] = (v[1::7].float() * 2.0 ** 10).to(v.dtype)
        k[5:9] = (k[5:9].float() * 8).to(k.dtype)
    b = Batch(dev, q_lens, kv_lens, 4, 2, 128, 16, 8, False, torch.bfloat16, edit=edit)
    b.check(b.run())

    def wide(q, k, v, cu):
        q *= 1e15
        k *= 1e-15
        v *= 1e25
    b = Batch(dev, q_lens, kv_lens, 4, 2, 128, 16, 8, True, torch.bfloat16, edit=wide)
    b.check(b.run(), "wide")

    def zeros(q, k, v, cu):
        q[0], k[3], v[1] = 0, 0, 0
    b = Batch(dev, q_lens, kv_lens, 4, 2, 128, 16, 4, True, torch.bfloat16, edit=zeros)
    b.check(b.run(), "zeros")

    def nothing(q, k, v, cu):
        v.zero_()
    b = Batch(dev, q_lens, kv_lens, 4, 2, 128, 16, 4, True, torch.bfloat16, edit=nothing)
    assert float(b.run().abs().max()) == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e30])
@pytest.mark.parametrize("q_len,kv_len", [(50, 50), (150, 170), (4, 90), (1, 64)])
def test_bad_values_reach_only_the_queries_that_see_them(dev, bad, q_len, kv_len):
    """Bad keys and values at positions that some queries of the tile do not see, and
    in slots past the end of the sequence."""
    for which in ("k", "v"):
        at = kv_len - (q_len + 1) // 2

        def edit(q, k, v, cu):
            (k if which == "k" else v)[at:] = bad

        b = Batch(dev, [q_len], [kv_len], 4, 2, 64, 16, 8, True, torch.bfloat16, edit=edit)
        clean = Batch(dev, [q_len], [kv_len], 4, 2, 64, 16, 8, True, torch.bfloat16)
        got = b.run()
        first = q_len - (kv_len - at)  # the first query that sees a bad key
        clean.check(torch.cat([got[:first], clean.run()[first:]]), f"{which} {bad}")
        if bad != 1e30:
            assert bool(got[first:].isnan().any(-1).all()), which
    # a sequence that ends before the bad slots of its last page
    b = Batch(dev, [q_len], [kv_len], 4, 2, 64, 16, 8, True, torch.bfloat16)
    ref = b.run()
    c = b.cache
    used = serving.slot_map(b.table, 16, [0, kv_len], [kv_len])
    for t in (c.k_scale, c.v_scale):
        flat = t.permute(0, 2, 1).reshape(-1, t.shape[1]).clone()
        keep = flat[used.to(dev)].clone()
        flat[:] = bad
        flat[used.to(dev)] = keep
        t.copy_(flat.view(t.shape[0], t.shape[2], t.shape[1]).permute(0, 2, 1))
    assert_bitexact(b.run(), ref, "slots past the end")


@pytest.mark.parametrize("q_len,kv_len", [(1, 100), (30, 100), (130, 200)])
def test_bad_pages_and_rows_outside(dev, q_len, kv_len):
    from g2ptq_amd import paged_attention
    b = Batch(dev, [q_len, q_len], [kv_len, kv_len], 4, 2, 64, 16, 8, True, torch.bfloat16)
    table = b.table.to(dev)
    lens = torch.tensor(b.kv_lens, dtype=torch.int32, device=dev)
    ref = b.run()
    # rows before the first and after the last sequence are zero
    q = torch.cat([b.q[:1]] * 3 + [b.q, b.q[:2]])
    out = paged_attention(q, b.cache, table, (offsets(b.q_lens) + 3).to(dev), lens)
    assert float(out[:3].abs().max()) == 0 and float(out[-2:].abs().max()) == 0
    b.check(out[3:-2], "shifted")
    # the second sequence's pages are not in the cache: the first is as it was
    for bad in (-1, 1 << 30):
        t = table.clone()
        t[1] = bad
        out = paged_attention(b.q, b.cache, t, offsets(b.q_lens).to(dev), lens)
        assert_bitexact(out[:q_len], ref[:q_len], "first")
        assert float(out[q_len:].abs().max()) == 0
        with pytest.raises(IndexError):
            b.cache.check()
    # a length beyond the table: the keys it has are attended
    lens2 = lens.clone()
    lens2[1] = 1 << 20
    out = paged_attention(b.q, b.cache, table, offsets(b.q_lens).to(dev), lens2)
    assert_bitexact(out[:q_len], ref[:q_len], "first")
    with pytest.raises(IndexError):
        b.cache.check()
    # no sequences, no tokens
    none = paged_attention(b.q, b.cache, table[:0], torch.zeros(1, dtype=torch.int32, device=dev),
                           lens[:0])
    assert float(none.abs().max()) == 0
    assert paged_attention(b.q[:0], b.cache, table, torch.zeros(3, dtype=torch.int32, device=dev),
                           lens).shape == (0, 4, 64)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [3000, 40]), ([100], [400])], ids=str)
def test_another_stream_and_a_graph(dev, q_lens, kv_lens):
    from g2ptq_amd import paged_attention
    b = Batch(dev, q_lens, kv_lens, 8, 2, 128, 16, 4, False, torch.bfloat16)
    ref = b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = b.run()
    torch.cuda.current_stream().wait_stream(side)
    assert_bitexact(out, ref, "stream")
    table, cu = b.table.to(dev), offsets(q_lens).to(dev)
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=dev)
    q = b.q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention(q, b.cache, table, cu, lens)
    for i in range(3):
        q.copy_(b.q * (i + 1))
        lens.copy_(torch.tensor([n - i for n in kv_lens]))
        graph.replay()
        torch.cuda.synchronize()
        assert_bitexact(out, paged_attention(q, b.cache, table, cu, lens), f"replay {i}")


def test_repeated_calls_give_the_same_bits(dev):
    b = Batch(dev, [1, 30], [5000, 2000], 8, 2, 128, 64, 8, False, torch.float16)
    ref = b.run()
    for _ in range(3):
        assert_bitexact(b.run(), ref, "again")


def test_refusals(dev):
    from g2ptq_amd import PagedKVCache, paged_attention
    cache = PagedKVCache(4, 16, 2, 64, device=dev)
    q = torch.zeros(3, 4, 64, device=dev, dtype=torch.float16)
    i32 = dict(dtype=torch.int32, device=dev)
    table, cu, lens = torch.zeros(1, 1, **i32), torch.tensor([0, 3], **i32), torch.tensor([3], **i32)
    with pytest.raises(NotImplementedError):
        paged_attention(q.float(), cache, table, cu, lens)
    with pytest.raises(ValueError, match="heads"):
        paged_attention(q[:, :3], cache, table, cu, lens)
    with pytest.raises(ValueError, match="queries of shape"):
        paged_attention(q[..., :32], cache, table, cu, lens)
    with pytest.raises(ValueError, match="cu_q"):
        paged_attention(q, cache, table, cu[:1], lens)
    with pytest.raises(ValueError, match="kv_lens"):
        paged_attention(q, cache, table, cu, lens.long())
    with pytest.raises(RuntimeError, match="GPU tensor"):
        paged_attention(q.cpu(), cache, table, cu, lens)
    with pytest.raises(RuntimeError, match="inference only"):
        paged_attention(q.clone().requires_grad_(), cache, table, cu, lens)
