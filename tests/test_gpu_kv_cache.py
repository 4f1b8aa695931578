"""GPU: the paged cache against the oracle: codes, scales and zero points bit for
bit, what reading gives back rounded once, over head sizes, bits, grids, types,
strides, page sizes and lengths; skipped slots, bad indices, refusals."""
import pytest
import torch

from oracle import serving
from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu


def make_batch(seed, lens, page, spare=3):
    """A page table for sequences of these lengths over shuffled pages, -1 past
    each sequence's last page, and the pool's size."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table, pool


def offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)


def values(T, H, D, dtype, seed):
    g = gen(seed)
    x = torch.randn(T, H, D, generator=g) * torch.exp(torch.randn(H, D, generator=g)) + 0.3
    return (x * torch.exp(torch.randn(T, 1, 1, generator=g))).to(dtype)


def unpack(codes, bits):
    if bits == 8:
        return codes.int()
    return torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).int()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("bits,sym", [(8, True), (8, False), (4, True), (4, False)])
@pytest.mark.parametrize("H,D,page", [(1, 16, 1), (3, 64, 16), (2, 80, 4), (8, 128, 64),
                                      (1, 256, 32), (5, 48, 128), (2, 32, 8), (1, 240, 4096)])
def test_written_codes_and_what_they_stand_for(dev, H, D, page, bits, sym, dtype):
    from g2ptq_amd import PagedKVCache
    lens = [5, 0, 1, page, page + 1, 17]
    table, pool = make_batch(page + D, lens, page)
    cache = PagedKVCache(pool, page, H, D, bits=bits, sym=sym, device=dev)
    T, cu = sum(lens), offsets(lens)
    k, v = values(T, H, D, dtype, 1), values(T, H, D, dtype, 2)
    slots = serving.slot_map(table, page, cu.tolist(), lens)
    cache.write(k.to(dev), v.to(dev), slots.to(dev))
    back = cache.read(table.to(dev), cu.to(dev), T, dtype=dtype)
    half = 2 ** (bits - 1)
    for x, codes, scale, zero, got in (
            (k, cache.k_codes, cache.k_scale, cache.k_zero, back[0]),
            (v, cache.v_codes, cache.v_scale, cache.v_zero, back[1])):
        rc, rs, rz = serving.quantize(x, bits, sym)
        at = (slots // page, slice(None), slots % page)
        assert_bitexact(scale.cpu()[at], rs, "scale")
        assert_bitexact(unpack(codes.cpu()[at], bits).float() - half, rc, "codes")
        if not sym:
            assert_bitexact(zero.cpu()[at].float() - half, rz, "zero")
        # one fp32 product, then one rounding to dtype: as torch rounds it
        assert_bitexact(got, (rs[..., None] * (rc - rz[..., None])).to(dtype), "read")
    cache.check()


def test_views_of_one_projection_and_odd_strides(dev):
    from g2ptq_amd import PagedKVCache
    H, D, page, T = 4, 64, 16, 50
    table, pool = make_batch(3, [T], page)
    cu = offsets([T])
    slots = serving.slot_map(table, page, [0, T], [T]).to(dev)
    big = values(T, 3 * H, D + 3, torch.bfloat16, 4).to(dev)
    for k, v in ((big[:, :H, :D], big[:, H:2 * H, 1:1 + D]),
                 (big[:, ::3, 3:], big.flip(0)[:, 2:6, :D]),
                 (big[:, :H, :D].transpose(0, 1).contiguous().transpose(0, 1),
                  big[:, :1, :D].expand(T, H, D))):
        a = PagedKVCache(pool, page, H, D, bits=4, sym=False, device=dev)
        b = PagedKVCache(pool, page, H, D, bits=4, sym=False, device=dev)
        a.write(k, v, slots)
        b.write(k.clone().contiguous(), v.clone().contiguous(), slots)
        for x, y in zip(a.read(table.to(dev), cu.to(dev), T), b.read(table.to(dev), cu.to(dev), T)):
            assert_bitexact(x, y, "strided")


def test_zero_and_bad_values_stay_in_their_token_and_head(dev):
    from g2ptq_amd import PagedKVCache
    H, D, page, T = 3, 128, 16, 20
    table, pool = make_batch(9, [T], page)
    cu = offsets([T]).to(dev)
    slots = serving.slot_map(table, page, [0, T], [T]).to(dev)
    for sym in (True, False):
        k = values(T, H, D, torch.float16, 5)
        k[3, 1], k[4, 0, 9], k[5, 2, 100], k[6, 1, 0] = 0, float("nan"), float("inf"), -float("inf")
        cache = PagedKVCache(pool, page, H, D, bits=8, sym=sym, device=dev)
        cache.write(k.to(dev), k.to(dev), slots)
        got = cache.read(table.to(dev), cu, T, dtype=torch.float32)[0].cpu()
        rc, rs, rz = serving.quantize(k, 8, sym)
        assert_bitexact(got, rs[..., None] * (rc - rz[..., None]), f"sym={sym}")
        for t, h in ((4, 0), (5, 2), (6, 1)):
            assert bool(got[t, h].isnan().all())
        assert float(got[3, 1].abs().max()) == 0
        assert int(got.isnan().sum()) == 3 * D


def test_skipped_slots_bad_indices_and_rows_outside(dev):
    from g2ptq_amd import PagedKVCache
    H, D, page, pool = 2, 64, 16, 4
    cache = PagedKVCache(pool, page, H, D, device=dev)
    k = values(6, H, D, torch.bfloat16, 6).to(dev)
    slots = torch.tensor([0, -1, 17, -5, 63, 2], device=dev)
    cache.write(k, k, slots)
    cache.check()
    table = torch.tensor([[0], [1], [3]], dtype=torch.int32, device=dev)
    # rows 0, 1 before the first sequence, the last two after the last
    cu = torch.tensor([2, 5, 7, 23], dtype=torch.int32, device=dev)
    got = cache.read(table, cu, 25)[0].float()
    rc, rs, rz = serving.quantize(k.cpu(), 8, True)
    ref = (rs[..., None] * rc).bfloat16().float().to(dev)
    full = torch.zeros(25, H, D, device=dev)
    full[2], full[4], full[6], full[22] = ref[0], ref[5], ref[2], ref[4]
    assert_bitexact(got, full, "rows")
    cache.check()
    before = [t.clone() for t in (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)]
    cache.write(k[:2], k[:2], torch.tensor([pool * page, 1 << 40], device=dev))
    with pytest.raises(IndexError):
        cache.check()
    cache.check()
    for a, b in zip(before, (cache.k_codes, cache.k_scale, cache.v_codes, cache.v_scale)):
        assert_bitexact(a, b, "untouched")
    for bad in (pool, -1, 1 << 30):
        t = table.clone()
        t[1, 0] = bad
        got = cache.read(t, cu, 25)[0].float()
        assert float(got[5:7].abs().max()) == 0
        with pytest.raises(IndexError):
            cache.check()
    # a sequence longer than its table row
    cu = torch.tensor([0, 18], dtype=torch.int32, device=dev)
    assert float(cache.read(table[:1], cu, 18)[0][16:].float().abs().max()) == 0
    with pytest.raises(IndexError):
        cache.check()
    k0, v0 = cache.read(table, torch.zeros(4, dtype=torch.int32, device=dev), 0)
    assert k0.shape == (0, H, D)
    cache.write(k[:0], k[:0], slots[:0])


def test_offsets_beyond_32_bits(dev):
    """A pool of more than 2^32 bytes of codes: the last page is the last page."""
    from g2ptq_amd import PagedKVCache
    H, D, page = 8, 256, 4096
    pool = (1 << 32) // (H * D * page) + 3
    cache = PagedKVCache(pool, page, H, D, device=dev)
    k, v = values(5, H, D, torch.bfloat16, 7), values(5, H, D, torch.bfloat16, 8)
    slots = torch.tensor([pool * page - 1, (pool - 1) * page, 0, pool * page - 2, 5])
    cache.write(k.to(dev), v.to(dev), slots.to(dev))
    table = torch.tensor([[pool - 1]], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, page], dtype=torch.int32, device=dev)
    gk, gv = cache.read(table, cu, page, dtype=torch.float32)
    for x, got in ((k, gk), (v, gv)):
        rc, rs, _ = serving.quantize(x, 8, True)
        ref = rs[..., None] * rc
        for i, p in ((0, page - 1), (1, 0), (3, page - 2)):
            assert_bitexact(got[p], ref[i], str(p))
        assert float(got[1:page - 2].abs().max()) == 0
    cache.check()


def test_another_stream_and_a_graph(dev):
    from g2ptq_amd import PagedKVCache
    H, D, page, T = 2, 128, 16, 40
    table, pool = make_batch(1, [T], page)
    cu = offsets([T]).to(dev)
    slots = serving.slot_map(table, page, [0, T], [T]).to(dev)
    table = table.to(dev)
    cache = PagedKVCache(pool, page, H, D, bits=4, sym=False, device=dev)
    k, v = (values(T, H, D, torch.bfloat16, s).to(dev) for s in (1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write(k, v, slots)
        got = cache.read(table, cu, T)
    torch.cuda.current_stream().wait_stream(side)
    rc, rs, rz = serving.quantize(k.cpu(), 4, False)
    assert_bitexact(got[0], (rs[..., None] * (rc - rz[..., None])).bfloat16(), "stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, slots)
        out = cache.read(table, cu, T)
    for i in range(3):
        k.copy_(values(T, H, D, torch.bfloat16, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        rc, rs, rz = serving.quantize(k.cpu(), 4, False)
        assert_bitexact(out[0], (rs[..., None] * (rc - rz[..., None])).bfloat16(), f"replay {i}")


def test_refusals(dev):
    from g2ptq_amd import PagedKVCache
    for args, kw in (((4, 16, 2, 64), {"bits": 3}), ((4, 12, 2, 64), {}), ((4, 16, 2, 72), {}),
                     ((4, 16, 2, 512), {}), ((4, 8192, 2, 64), {}), ((4, 16, 0, 64), {})):
        with pytest.raises(ValueError):
            PagedKVCache(*args, device=dev, **kw)
    cache = PagedKVCache(4, 16, 2, 64, device=dev)
    k = torch.zeros(3, 2, 64, device=dev)
    slots = torch.zeros(3, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="keys of shape"):
        cache.write(k[:, :1], k, slots)
    with pytest.raises(ValueError, match="slots"):
        cache.write(k, k, slots.int())
    with pytest.raises(ValueError, match="3 keys"):
        cache.write(k, k, slots[:2])
    with pytest.raises(NotImplementedError):
        cache.write(k, k.half(), slots)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        cache.write(k.cpu(), k, slots)
    with pytest.raises(RuntimeError, match="inference only"):
        cache.write(k.clone().requires_grad_(), k, slots)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="cu_tokens"):
        cache.read(table, torch.zeros(3, dtype=torch.int32, device=dev), 1)
    with pytest.raises(ValueError, match="table"):
        cache.read(table.long(), torch.zeros(2, dtype=torch.int32, device=dev), 1)
    with pytest.raises(NotImplementedError):
        cache.read(table, torch.zeros(2, dtype=torch.int32, device=dev), 1, dtype=torch.float64)


def test_a_caches_tensors_are_not_replaced(dev):
    """The kernels know them by their addresses."""
    from g2ptq_amd import PagedKVCache
    c = PagedKVCache(2, 16, 1, 16, device=dev)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale", "k_zero", "v_zero", "flags"):
        with pytest.raises(AttributeError):
            setattr(c, name, torch.zeros(1, device=dev))
    c.k_scale.fill_(1.0)
    k, v = c.read(torch.zeros(1, 1, dtype=torch.int32, device=dev),
                  torch.tensor([0, 3], dtype=torch.int32, device=dev), 3, torch.float32)
    assert bool((k == -128).all()) and bool((v == 0).all())
