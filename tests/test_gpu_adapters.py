"""GPU: low-rank adapters of many requests against the formula in 64 bits: ranks, ragged sizes,
tokens in any order, none, strides, extreme values, in place; refusals."""
import pytest
import torch

from oracle import layer_ops
from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


class Set:
    def __init__(self, dev, ranks, N, K, dtype, seed=1, scale=None):
        from g2ptq_amd import LowRankAdapters
        g = gen(seed)
        self.down = [(torch.randn(r, K, generator=g) / K ** 0.5).to(dtype) for r in ranks]
        self.up = [(torch.randn(N, r, generator=g) / r ** 0.5).to(dtype) for r in ranks]
        self.scale = [0.25 + 0.5 * i for i in range(len(ranks))] if scale is None else scale
        self.dev, self.dtype, self.N, self.K, self.g = dev, dtype, N, K, g
        self.own = LowRankAdapters([d.to(dev) for d in self.down], [u.to(dev) for u in self.up],
                                   scale=self.scale)

    def x(self, T):
        x = torch.randn(T, self.K, generator=self.g)
        return (x * torch.exp(0.5 * torch.randn(T, 1, generator=self.g))).to(self.dtype)

    def base(self, T):
        return torch.randn(T, self.N, generator=self.g).to(self.dtype)

    def index(self, T, kind):
        n = len(self.down)
        if kind == "sorted":
            return torch.sort(torch.randint(-1, n, (T,), generator=self.g))[0].int()
        if kind == "one":
            return torch.full((T,), n - 1, dtype=torch.int32)
        if kind == "none":
            return torch.full((T,), -5, dtype=torch.int32)
        return torch.randint(-1, n, (T,), generator=self.g).int()

    def check(self, y, x, index, base):
        ref, err = layer_ops.adapters(x, index, self.down, self.up, self.scale, base)
        bound = layer_ops.rounded(self.dtype, ref, err)
        assert y.dtype is self.dtype and y.shape == ref.shape
        off = (y.cpu().double() - ref).abs()
        assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
        if base is not None:
            assert_bitexact(y.cpu()[index < 0], base[index < 0], "tokens without an adapter")

    def run(self, T, kind):
        dev, x, index, base = self.dev, self.x(T), self.index(T, kind), self.base(T)
        y = self.own(x.to(dev), index.to(dev), base=base.to(dev))
        self.check(y, x, index, base)
        self.check(self.own(x.to(dev), index.to(dev)), x, index, None)
        z = base.to(dev)
        assert self.own.add_(z, x.to(dev), index.to(dev)) is z
        assert_bitexact(z, y, "in place")
        self.own.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("ranks,N,K", [
    ([1], 1, 1), ([16], 64, 64), ([8, 16, 3], 100, 70), ([24, 12], 300, 515), ([32], 257, 2752),
    ([48, 17, 64], 130, 384), ([64] * 4, 512, 1040), ([65, 16, 128, 200], 96, 300),
    ([512, 1], 72, 130), ([16] * 80, 64, 96)], ids=lambda v: str(v)[:24])
def test_adapters_are_the_formula(dev, ranks, N, K, dtype):
    s = Set(dev, ranks, N, K, dtype)
    for T in (1, 2, 15, 16, 17, 63, 64, 65, 130, 333):
        for kind in ("random", "sorted", "one"):
            s.run(T, kind)
    s.run(70, "none")


@pytest.mark.parametrize("n", [2, 7, 20, 40])
def test_requests_of_any_length(dev, n):
    """Prompts of as many tokens as there are adapters and about, adapters that come again, and
    tokens without one between them."""
    s = Set(dev, [16, 24] * (n // 2) + [8] * (n % 2), 96, 130, torch.bfloat16)
    for length in (1, n - 1, n, n + 1, 2 * (n + 1), 32):
        of = torch.arange(1 + 200 // length) % n
        mixed = torch.randint(-1, n, (len(of),), generator=s.g)
        for order in (of, of.flip(0), mixed, mixed * (torch.arange(len(of)) % 2) - 1 * (mixed < 0)):
            index = order.repeat_interleave(length)[:200].int()
            T = len(index)
            x, base = s.x(T), s.base(T)
            s.check(s.own(x.to(dev), index.to(dev), base=base.to(dev)), x, index, base)


@pytest.mark.parametrize("T", [1, 48, 64, 2000])
def test_more_columns_than_one_workgroup_takes(dev, T):
    for dtype in DTYPES:
        s = Set(dev, [16, 40], 200, 8200, dtype)
        s.run(T, "random")
        s.run(T, "sorted")


@pytest.mark.parametrize("T", [600, 5000, 70000])
def test_many_tokens(dev, T):
    s = Set(dev, [16, 8, 30], 72, 136, torch.bfloat16)
    s.run(T, "sorted")
    s.run(T, "random")


def test_rows_that_no_cache_holds(dev):
    """From 2^26 outputs on rows are streamed past the caches: the same bits as in parts."""
    T, N = 70000, 1000
    s = Set(dev, [16, 40, 64, 9], N, 72, torch.bfloat16)
    g = torch.Generator(dev).manual_seed(1)
    x = torch.randn(T, 72, generator=g, device=dev).bfloat16()
    base = torch.randn(T, N, generator=g, device=dev).bfloat16()
    index = torch.arange(-1, 4, device=dev).repeat_interleave(T // 5).int()
    index[:3000] = torch.randint(-1, 4, (3000,), generator=g, device=dev)
    y = s.own(x, index, base=base)
    z = base.clone()
    s.own.add_(z, x, index)
    assert_bitexact(z, y, "in place")
    for at in range(0, T, 10000):
        part = slice(at, at + 10000)
        assert_bitexact(s.own(x[part], index[part], base=base[part]), y[part], f"rows from {at}")
    s.check(y[-500:], x[-500:].cpu(), index[-500:].cpu(), base[-500:].cpu())


def test_more_windows_than_a_launch_takes(dev):
    """2^27 tokens and some: the last windows lie past the first launch."""
    T = (1 << 27) + 100
    s = Set(dev, [4], 8, 8, torch.float16)
    x = torch.zeros(T, 8, dtype=torch.float16, device=dev)
    index = torch.full((T,), -1, dtype=torch.int32, device=dev)
    x[-70:], index[-70:] = s.x(70).to(dev), 0
    y = s.own(x, index)
    s.check(y[-70:], x[-70:].cpu(), index[-70:].cpu(), None)
    assert not bool(y[:1 << 20].any()) and not bool(y[-(1 << 20):-70].any())
    del x, y
    torch.cuda.empty_cache()


def test_tokens_do_not_depend_on_their_neighbours(dev):
    """A token's row has the same bits with other tokens around it, in any order."""
    s = Set(dev, [16, 24, 64], 200, 300, torch.bfloat16)
    x, index, base = s.x(60).to(dev), s.index(60, "random").to(dev), s.base(60).to(dev)
    y = s.own(x, index, base=base)
    order = torch.randperm(60, generator=gen(3)).to(dev)
    assert_bitexact(s.own(x[order], index[order], base=base[order]), y[order], "order")
    assert_bitexact(s.own(x[7:55], index[7:55], base=base[7:55]), y[7:55], "part")
    for _ in range(3):
        assert_bitexact(s.own(x, index, base=base), y, "again")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rank,K,N", [(16, 4096, 3000), (40, 4095, 1030), (64, 2752, 520),
                                      (200, 1500, 300), (16, 14336, 64)])
def test_bits_go_by_the_number_of_tokens_alone(dev, dtype, rank, K, N):
    """At the same number of tokens a token's row has the same bits wherever it stands and however
    many of the tokens around it share its adapter."""
    T = 150
    s = Set(dev, [rank, 16, rank], N, K, dtype)
    probes = torch.tensor([0, 2, 0])
    px, pbase, x, base = (v.to(dev) for v in (s.x(3), s.base(3), s.x(T), s.base(T)))
    want = None
    for at in (0, 14, 62, 70, 128, 147):
        for sharers in (0, 1, 13, 14, 20, 61, T):
            index = torch.ones(T, dtype=torch.int32)
            index[:min(T, at // 64 * 64 + sharers)] = 0
            index[at:at + 3] = probes.int()
            xs, bases = x.clone(), base.clone()
            xs[at:at + 3], bases[at:at + 3] = px, pbase
            y = s.own(xs, index.to(dev), base=bases)
            want = y[at:at + 3].clone() if want is None else want
            assert_bitexact(y[at:at + 3], want, f"from {at} with {sharers} sharers")
            s.own.add_(bases, xs, index.to(dev))
            assert_bitexact(bases, y, "in place")
    s.check(want, px.cpu(), probes, pbase.cpu())


@pytest.mark.parametrize("K,N", [(1, 1), (3, 7), (7, 9), (63, 65), (65, 127), (129, 190), (191, 64),
                                 (1023, 129), (2049, 33)])
@pytest.mark.parametrize("T,ranks", [(5, [16]), (70, [16, 40]), (130, [33, 64, 3])])
def test_rows_at_any_address(dev, K, N, T, ranks):
    """Rows that start between words or inside a piece of eight values, NaN on every side."""
    for dtype in DTYPES:
        s = Set(dev, ranks, N, K, dtype)
        x, base, index = s.x(T).to(dev), s.base(T).to(dev), s.index(T, "random").to(dev)

        def inside(v, before, behind):
            wide = torch.full((T, before + v.shape[1] + behind), float("nan"), dtype=dtype, device=dev)
            wide[:, before:before + v.shape[1]] = v
            return wide, wide[:, before:before + v.shape[1]]

        # (rows of whole pieces at aligned addresses)
        ref = s.own(inside(x, 8, 16 - K % 8)[1], index, base=inside(base, 8, 16 - N % 8)[1])
        assert not ref.isnan().any()
        for before, behind in ((1, 0), (0, 1), (1, 1), (2, 0), (3, 2), (8, 7)):
            xw, xv = inside(x, before, behind)
            bw, bv = inside(base, before, behind)
            assert_bitexact(s.own(xv, index, base=bv), ref, f"{before} {behind}")
            kept = bw.clone()
            s.own.add_(bv, xv, index)
            assert_bitexact(bv, ref, f"{before} {behind} in place")
            kept[:, before:before + N] = ref
            assert torch.equal(bw.view(torch.int16), kept.view(torch.int16))


def test_strides_and_shapes(dev):
    for dtype in DTYPES:
        s = Set(dev, [16, 24], 70, 90, dtype)
        x, base, index = s.x(24), s.base(24), s.index(24, "random")
        ref = s.own(x.to(dev), index.to(dev), base=base.to(dev))
        wide = torch.zeros(24, 200, dtype=dtype, device=dev)
        wide[:, 5:95], wide[:, 101:171] = x.to(dev), base.to(dev)
        xv, bv = wide[:, 5:95], wide[:, 101:171]
        assert_bitexact(s.own(xv, index.to(dev), base=bv), ref, "views")
        assert_bitexact(s.own(x.t().contiguous().t().to(dev), torch.stack([index] * 2, 1).to(dev)[:, 0],
                              base=base.t().contiguous().to(dev).t()), ref, "transposed")
        three = s.own(x.to(dev).view(2, 12, 90), index.to(dev).view(2, 12),
                      base=base.to(dev).view(2, 12, 70))
        assert three.shape == (2, 12, 70)
        assert_bitexact(three.view(24, 70), ref, "three dimensions")
        one = s.own(x[3].to(dev), index[3].to(dev), base=base[3].to(dev))
        assert one.shape == (70,)
        assert_bitexact(one, ref[3], "one token")
        assert s.own(x[:0].to(dev), index[:0].to(dev)).shape == (0, 70)
        rest = wide.clone()
        s.own.add_(wide[:, 101:171], xv, index.to(dev))
        assert_bitexact(wide[:, 101:171], ref, "in place")
        wide[:, 101:171] = rest[:, 101:171]
        assert_bitexact(wide, rest, "around")
        same = x[:1].to(dev).expand(24, 90)
        assert_bitexact(s.own(same, index.to(dev)), s.own(same.contiguous(), index.to(dev)), "expanded")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("size", [1e-6, 3e-3, 300.0, 30000.0])
def test_small_and_large_inner_values(dev, dtype, size):
    """h far below and above fp16's range: rows keep their precision."""
    s = Set(dev, [16, 40], 64, 128, dtype, scale=[1e-3, 1e3])
    s.down = [(d.double() * size).to(dtype) for d in s.down]
    from g2ptq_amd import LowRankAdapters
    s.own = LowRankAdapters([d.to(dev) for d in s.down], [u.to(dev) for u in s.up], scale=s.scale)
    x, index = s.x(40), s.index(40, "random")
    if dtype is torch.float16 and size > 100:  # (outputs within fp16's range)
        s.up = [(u.double() / size / 1e3).to(dtype) for u in s.up]
        s.own = LowRankAdapters([d.to(dev) for d in s.down], [u.to(dev) for u in s.up],
                                scale=s.scale)
    s.check(s.own(x.to(dev), index.to(dev)), x, index, None)


def test_nan_and_infinities_stay_in_their_tokens(dev):
    """An infinite input makes its token's row what the formula makes of it; others keep their
    bits, and so do the bases of tokens without an adapter."""
    for dtype in DTYPES:
        s = Set(dev, [16, 20], 48, 100, dtype)
        x, base = s.x(30), s.base(30)
        index = s.index(30, "random")
        index[:4] = torch.tensor([0, 1, 1, -1])
        clean = s.own(x.to(dev), index.to(dev), base=base.to(dev)).cpu()
        x[0, 3], x[1, 4], x[2, 99], x[3] = float("inf"), float("nan"), -float("inf"), float("nan")
        y = s.own(x.to(dev), index.to(dev), base=base.to(dev)).cpu()
        assert_bitexact(y[3:], clean[3:], "others")
        assert bool(y[1].isnan().all())
        for t in (0, 2):
            h = x[t].double() @ s.down[int(index[t])].double().T
            ref = base[t].double() + s.scale[int(index[t])] * (s.up[int(index[t])].double() @ h)
            assert bool((y[t].isnan() == ref.isnan()).all())
            assert bool((y[t][~ref.isnan()].double() == ref[~ref.isnan()]).all())
    s.own.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("ranks,N", [([16, 5], 70), ([20, 33], 264), ([64, 80], 130), ([200, 16], 65)])
def test_infinite_and_nan_weights(dev, dtype, ranks, N):
    """Weights that are infinite or NaN: rows are what the formula makes of them, in their own
    channels and their own adapter's tokens."""
    K, T = 100, 90
    clean = Set(dev, ranks, N, K, dtype)
    s = Set(dev, ranks, N, K, dtype)
    inf, nan = float("inf"), float("nan")
    s.up[0][3, 1], s.up[0][40, ranks[0] - 1], s.up[0][N - 1, 0], s.up[0][5, 2] = inf, -inf, inf, nan
    s.up[0][7, 0], s.up[0][7, 1] = inf, -inf
    s.up[0][9, 0], s.up[0][9, 1] = -inf, -inf
    from g2ptq_amd import LowRankAdapters
    s.own = LowRankAdapters([d.to(dev) for d in s.down], [u.to(dev) for u in s.up], scale=s.scale)
    x, base = s.x(T), s.base(T)
    x[4, 2], x[5] = inf, 0
    for index in (s.index(T, "random"), torch.zeros(T, dtype=torch.int32)):
        index[4:6] = 0
        y = s.own(x.to(dev), index.to(dev), base=base.to(dev)).cpu()
        whole = clean.own(x.to(dev), index.to(dev), base=base.to(dev)).cpu()
        touched = torch.zeros(T, N, dtype=torch.bool)
        touched[(index == 0)[:, None] & torch.tensor([c in (3, 5, 7, 9, 40, N - 1)
                                                      for c in range(N)])[None]] = True
        assert_bitexact(y[~touched], whole[~touched], "others")
        for t in (index == 0).nonzero()[:, 0].tolist():
            h = x[t].double() @ s.down[0].double().T
            # (rounded as the kernel holds it, an infinity or a zero is one of the formula's)
            ref = base[t].double() + s.scale[0] * (s.up[0].double() @ h)
            for c in (3, 5, 7, 9, 40, N - 1):
                a, b = float(y[t, c]), float(ref[c])
                assert a == b or (a != a and b != b), (t, c, a, b)


def test_inner_values_next_to_the_largest(dev):
    """An h between the largest bf16 and the largest fp32 is no infinity."""
    from g2ptq_amd import LowRankAdapters
    top = torch.finfo(torch.bfloat16).max
    down = torch.zeros(3, 40, dtype=torch.bfloat16)
    down[:, 0], down[0, 1], down[1, 1], down[2, 1] = top, 2.0 ** 119, 1.5 * 2.0 ** 119, -2.0 ** 119
    down[1] *= -1
    up = torch.zeros(20, 3, dtype=torch.bfloat16)
    up[:3] = torch.eye(3) * 2.0 ** -20
    x = torch.ones(2, 40, dtype=torch.bfloat16)
    y = LowRankAdapters([down.to(dev)], [up.to(dev)])(x.to(dev), torch.zeros(2, dtype=torch.int32,
                                                                            device=dev))
    ref = x.double() @ down.double().T @ up.double().T
    # (all sums are exact: h has 8 bits more than bf16, and the result is rounded once)
    assert_bitexact(y, ref.bfloat16(), "result")


def test_an_index_of_no_adapter_is_flagged(dev):
    s = Set(dev, [16, 8], 40, 50, torch.bfloat16)
    x, base = s.x(100), s.base(100)
    index = s.index(100, "random")
    index[70] = 2
    y = s.own(x.to(dev), index.to(dev), base=base.to(dev))
    with pytest.raises(IndexError, match="2 adapters"):
        s.own.check()
    s.own.check()
    index[70] = -1
    s.check(y, x, index, base)


def test_adapters_beside_an_8_bit_linear(dev):
    from g2ptq_amd import Int8Linear
    s = Set(dev, [16, 8], 70, 130, torch.bfloat16)
    g = gen(9)
    lin = Int8Linear(torch.randint(-128, 128, (70, 130), generator=g, dtype=torch.int8).to(dev),
                     (torch.rand(70, generator=g) * 1e-3).to(dev))
    x, index = s.x(33), s.index(33, "random")
    y = lin(x.to(dev))
    s.check(s.own(x.to(dev), index.to(dev), base=y), x, index, y.cpu())


def test_replayed_graphs_do_not_share_workspaces(dev):
    s = Set(dev, [16, 24], 70, 600, torch.bfloat16)
    xs = [s.x(T).to(dev) for T in (20, 300)]
    idx = [s.index(len(x), "random").to(dev) for x in xs]
    want = [s.own(x, i) for x, i in zip(xs, idx)]
    graphs = []
    for x, i in zip(xs, idx):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = s.own(x, i)
        graphs.append((graph, out))
    for _ in range(4):
        for graph, _ in graphs:
            graph.replay()
        s.own(s.x(500).to(dev), s.index(500, "random").to(dev))
        torch.cuda.synchronize()
        for (_, out), ref in zip(graphs, want):
            assert_bitexact(out, ref, "replay")
            out.zero_()


def test_adapter_refusals(dev):
    from g2ptq_amd import LowRankAdapters
    d, u = torch.ones(4, 32, device=dev).half(), torch.ones(24, 4, device=dev).half()
    for err, args in ((ValueError, ([], [])), (ValueError, ([d], [u, u])),
                      (ValueError, ([d], [u[:, :3]])), (ValueError, ([d, d[:, :31]], [u, u])),
                      (ValueError, ([d, d.bfloat16()], [u, u])), (ValueError, ([d], [u.cpu()])),
                      (ValueError, ([d[:0]], [u[:, :0]])), (ValueError, ([d[0]], [u])),
                      (NotImplementedError, ([d.float()], [u.float()])),
                      (RuntimeError, ([d.cpu()], [u.cpu()])),
                      (ValueError, ([d], [u], [1.0, 2.0])),
                      (ValueError, ([torch.ones(513, 32, device=dev).half()],
                                    [torch.ones(24, 513, device=dev).half()]))):
        with pytest.raises(err):
            LowRankAdapters(*args)
    a = LowRankAdapters([d], [u], scale=0.5)
    x, i = torch.ones(3, 32, device=dev).half(), torch.zeros(3, dtype=torch.int32, device=dev)
    y = torch.ones(3, 24, device=dev).half()
    for err, call in ((ValueError, lambda: a(x, i.long())), (ValueError, lambda: a(x, i[:2])),
                      (ValueError, lambda: a(x[:, :31], i)), (ValueError, lambda: a(x, i.cpu())),
                      (NotImplementedError, lambda: a(x.float(), i)),
                      (NotImplementedError, lambda: a(x, i, base=y.float())),
                      (ValueError, lambda: a(x, i, base=y[:2])),
                      (ValueError, lambda: a(x, i, base=y[:, :3])), (RuntimeError, lambda: a(x.cpu(), i)),
                      (RuntimeError, lambda: a(x.clone().requires_grad_(), i)),
                      (RuntimeError, lambda: a(x, i, base=y.clone().requires_grad_())),
                      (ValueError, lambda: a.add_(y[:2], x, i)),
                      (ValueError, lambda: a.add_(y[:1].expand(3, 24), x, i)),
                      (ValueError, lambda: a.add_(y.t().contiguous().t(), x, i))):
        with pytest.raises(err):
            call()
    assert_bitexact(a(x, i), torch.full((3, 24), 64.0).half(), "result")
