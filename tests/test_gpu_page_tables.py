"""GPU: page tables and slot maps against lists of whole numbers: growth, release and its undoing
of a step, requests that do not fit, padding, rows named twice, long batches; the cache and its
attention on what they give; replayed graphs."""
import random

import pytest
import torch

from oracle import layer_ops
from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu


class Both:
    """The tables and the oracle, in step."""

    def __init__(self, dev, pages, page, seqs, width):
        from g2ptq_amd import PageTables
        self.dev, self.ref = dev, layer_ops.Pages(pages, page, seqs, width)
        self.own = PageTables(pages, page, seqs, width, device=dev)

    def i32(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.dev)

    def state(self):
        own, ref = self.own, self.ref
        n = int(own.free_count)
        assert n == len(ref.free) and own.free_pages[:n].tolist() == ref.free
        assert own.lengths.tolist() == ref.lengths and own.table.tolist() == ref.table()
        assert bool((own._mark == 0x7fffffff).all())

    def extend(self, rows, new, total=None):
        total = sum(n for n in new if n > 0) if total is None else total
        step = self.own.extend(self.i32(rows), self.i32(new), total)
        want = self.ref.extend(rows, new, total)
        for name, a, b in zip(step._fields, step, want):
            assert a.tolist() == b, name
        assert step.slots.dtype is step.positions.dtype is torch.int64
        self.state()
        return step

    def release(self, rows, keep=None):
        self.own.release(self.i32(rows), None if keep is None else self.i32(keep))
        self.ref.release(rows, keep)
        self.state()

    def check(self):
        bad, full = self.ref.bad, self.ref.full
        self.ref.bad = self.ref.full = False
        if bad or full:
            with pytest.raises(IndexError if bad else RuntimeError):
                self.own.check()
        self.own.check()


@pytest.mark.parametrize("page", [1, 2, 16, 64, 4096])
def test_requests_come_grow_and_go(dev, page):
    b = Both(dev, 4000 // page + 40, page, 12, 900 // page + 2)
    b.extend([3], [1])
    b.extend([3, 5, 0], [page, 3 * page + 1, 0])
    b.extend([0, 1], [17, 1], total=40)
    b.extend([5, 3], [1, 2])
    b.release([3])
    b.extend([7, 3], [5, 7 * page])
    b.release([5, 0], [2, 17])
    b.release([7, 5], [5, 0])
    b.extend([11, 5, 0, 3, 1, 7], [1] * 6)
    b.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_steps(dev, seed):
    """Ragged steps with requests that do not fit, padding, rows of no table and rows twice."""
    r = random.Random(seed)
    page = r.choice([1, 4, 16, 128])
    b = Both(dev, r.randint(5, 60), page, 20, r.randint(2, 9))
    for _ in range(25):
        n = r.randint(1, 14)
        rows = [r.randint(0, 19) for _ in range(n)] if r.random() < 0.3 else r.sample(range(20), n)
        rows = [-1 if r.random() < 0.1 else 20 + r.randint(0, 5) if r.random() < 0.03 else x
                for x in rows]
        if r.random() < 0.7:
            new = [r.choice([0, 1, 1, r.randint(0, 3 * page), -2 if r.random() < 0.1 else 1])
                   for _ in rows]
            total = sum(x for x in new if x > 0)
            b.extend(rows, new, r.choice([total, total, total + 9, max(0, total - 3)]))
        else:
            keep = None if r.random() < 0.4 else [
                r.choice([0, max(0, b.ref.lengths[x % 20] - r.randint(0, page)),
                          b.ref.lengths[x % 20] + (r.random() < 0.1)]) for x in rows]
            b.release(rows, keep)
        b.check()


@pytest.mark.parametrize("B", [1, 63, 64, 65, 1023, 1024, 1025, 3000, 4090, 4096, 4097, 5000])
def test_batches_of_any_length(dev, B):
    r = random.Random(B)
    b = Both(dev, 4 * B + 10, 4, B + 7, 6)
    rows = r.sample(range(B + 7), B)
    b.extend(rows, [r.randint(0, 5) for _ in rows])
    b.extend(rows[::-1], [r.choice([0, 1, 9]) for _ in rows], total=9 * B + 5)
    b.release(rows[::2], [min(3, b.ref.lengths[x]) for x in rows[::2]])
    b.extend(rows, [1] * B)
    b.release(rows[:B // 2 + 1])
    again = rows + rows[:3]
    b.extend(again, [2] * len(again))
    b.check()


@pytest.mark.parametrize("B,width,new", [(3, 5, 40), (40, 500, 3), (900, 40, 30), (5, 3000, 9000)])
def test_release_undoes_a_step(dev, B, width, new):
    """Each side of the size up to which one launch does all."""
    from g2ptq_amd import PageTables
    t = PageTables(2 * B * (new // 16 + 2), 16, 2 * B, width, device=dev)
    g = gen(B)
    rows = torch.randperm(2 * B, generator=g)[:B].int().to(dev)
    some = torch.randint(0, new // 2 + 1, (B,), generator=g).int()
    t.extend(rows, some.to(dev), int(some.sum()))
    t.release(rows[::3].contiguous())
    held = t.lengths[rows.long()].clone()
    before = [x.clone() for x in t._held]
    counts = torch.randint(0, new // 2 + 1, (B,), generator=g).int()
    first = t.extend(rows, counts.to(dev), int(counts.sum()))
    t.release(rows, held)
    for x, y in zip(t._held, before):
        assert_bitexact(x, y, "state")
    for x, y in zip(t.extend(rows, counts.to(dev), int(counts.sum())), first):
        assert_bitexact(x, y, "step")
    slots = first.slots[first.slots >= 0]
    assert len(slots) == int(counts.sum()) == len(slots.unique())
    t.check()


def test_large_step(dev):
    """A long prompt and many short ones: every slot once, in its request's pages."""
    from g2ptq_amd import PageTables
    B, page = 500, 64
    new = [300000] + [(i * 37) % 400 for i in range(B - 1)]
    t = PageTables(12000, page, B, 5000, device=dev)
    rows = torch.arange(B, dtype=torch.int32, device=dev)
    total = sum(new)
    s = t.extend(rows, torch.tensor(new, dtype=torch.int32, device=dev), total + 3)
    t.check()
    assert s.slots[-3:].tolist() == [-1] * 3 and len(s.slots[:-3].unique()) == total
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).to(dev)
    pos = torch.arange(total, device=dev) - s.cu.long()[seq]
    assert_bitexact(s.positions[:-3], pos, "positions")
    assert_bitexact(s.slots[:-3], s.table.long()[seq, pos // page] * page + pos % page, "slots")
    assert_bitexact(s.kv_lens, torch.tensor(new, dtype=torch.int32), "lengths")


def test_without_requests_tokens_or_pages(dev):
    from g2ptq_amd import PageTables
    b = Both(dev, 0, 8, 2, 3)
    b.extend([], [])
    b.extend([], [], total=5)
    b.extend([0, 1], [0, 0], total=2)
    b.release([])
    b.extend([0], [3])
    b.check()
    t = PageTables(2, 8, 2, 3, device=dev)
    rows = torch.tensor([0, 9, 1, 9], dtype=torch.int32, device=dev)[::2]
    assert not rows.is_contiguous()
    s = t.extend(rows, torch.tensor([3, 2], dtype=torch.int32, device=dev), 5)
    assert s.slots.tolist() == [0, 1, 2, 8, 9]


def test_page_tables_of_a_served_cache(dev):
    """Attention over a cache filled through the tables is what it is over pages in order."""
    from g2ptq_amd import PagedKVCache, PageTables, paged_attention
    H, D, page, lens = 2, 64, 16, [70, 5, 33]
    g = gen(1)
    k, v = (torch.randn(sum(lens), H, D, generator=g).half().to(dev) for _ in range(2))
    q = torch.randn(len(lens), 4, D, generator=g).half().to(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    cache, flat = (PagedKVCache(20, page, H, D, bits=8, device=dev) for _ in range(2))
    t = PageTables(cache.num_pages, page, 8, 6, device=dev)
    t.extend(torch.tensor([7, 2], **i32), torch.tensor([40, 20], **i32), 60)
    t.release(torch.tensor([2], **i32))
    rows = torch.tensor([4, 0, 6], **i32)
    for part in ([60, 4, 1], [10, 1, 32]):  # in two chunks
        at = t.lengths[rows.long()].tolist()
        s = t.extend(rows, torch.tensor(part, **i32), sum(part))
        first = [sum(lens[:i]) + n for i, n in enumerate(at)]
        take = torch.cat([torch.arange(f, f + n) for f, n in zip(first, part)]).to(dev)
        cache.write(k[take], v[take], s.slots)
    out = paged_attention(q, cache, s.table, torch.arange(4, **i32), s.kv_lens)
    t.check()
    cache.check()
    table = torch.tensor([[0, 1, 2, 3, 4], [5, 0, 0, 0, 0], [6, 7, 8, 0, 0]], **i32)
    slots = torch.cat([table[i].long().repeat_interleave(page)[:n] * page
                       + torch.arange(n, device=dev) % page for i, n in enumerate(lens)])
    flat.write(k, v, slots)
    ref = paged_attention(q, flat, table, torch.arange(4, **i32), torch.tensor(lens, **i32))
    assert_bitexact(out, ref, "attention")


def test_replayed_steps_take_their_own_pages(dev):
    from g2ptq_amd import PageTables
    rows = torch.tensor([1, 3], dtype=torch.int32, device=dev)
    new = torch.tensor([1, 5], dtype=torch.int32, device=dev)
    t = PageTables(40, 4, 4, 10, device=dev)
    ref = PageTables(40, 4, 4, 10, device=dev)
    t.extend(rows, new, 6)
    t.release(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = t.extend(rows, new, 6)
    for i in range(5):
        graph.replay()
        want = ref.extend(rows, new, 6)
        torch.cuda.synchronize()
        for a, b in zip(step, want):
            assert_bitexact(a, b, f"replay {i}")
        for a, b in zip(t._held, ref._held):
            assert_bitexact(a, b, f"state {i}")
        torch.ones(1 << 20, device=dev).sum().item()


def test_page_table_refusals(dev):
    from g2ptq_amd import PageTables
    for args in ((4, 3, 2, 2), (4, 8192, 2, 2), (-1, 8, 2, 2), (4, 8, 0, 2), (4, 8, 2, 0),
                 (4, 4096, 2, 1 << 20), (1 << 31, 8, 2, 2)):
        with pytest.raises(ValueError):
            PageTables(*args, device=dev)
    with pytest.raises(RuntimeError):
        PageTables(4, 8, 2, 2, device="cpu")
    t = PageTables(4, 8, 2, 2, device=dev)
    i = torch.zeros(2, dtype=torch.int32, device=dev)
    for call in (lambda: t.extend(i.long(), i, 4), lambda: t.extend(i, i.long(), 4),
                 lambda: t.extend(i, i[:1], 4), lambda: t.extend(i[None], i, 4),
                 lambda: t.extend(i.cpu(), i, 4), lambda: t.extend(i, i, -1),
                 lambda: t.extend(i, i, 1 << 31), lambda: t.release(i, i[:1]),
                 lambda: t.release(i.long()), lambda: t.release(i, i.cpu())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(AttributeError):
        t.table = i


def test_overwritten_state_stays_within_its_memory(dev):
    """Lengths and counts are the caller's to see; what no call can have left there is clamped."""
    from g2ptq_amd import PageTables
    t = PageTables(6, 8, 3, 4, device=dev)
    rows = torch.arange(3, dtype=torch.int32, device=dev)
    around = [x.clone() for x in t._held]
    t.lengths.copy_(torch.tensor([2 ** 31 - 1, -5, 40], dtype=torch.int32))
    t.free_count.fill_(1000)
    s = t.extend(rows, torch.ones(3, dtype=torch.int32, device=dev), 3)
    assert s.kv_lens.tolist() == [32, 1, 32] and s.slots.tolist()[::2] == [-1, -1]
    assert int(s.slots[1]) == 0 and t.free_count.tolist() == [5]
    t.release(rows)
    assert t.lengths.tolist() == [0, 0, 0] and bool((t.table == -1).all())
    assert 0 <= int(t.free_count) and [len(x) for x in t._held] == [len(x) for x in around]
    with pytest.raises(RuntimeError):
        t.check()
