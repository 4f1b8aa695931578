"""GPU: 8-bit linears against the oracle: token codes, scales and zero points bit
for bit, products within the rounding of fp32 scaling and of the output type,
at ragged sizes, strides, zero and non-finite rows; refusals."""
import pytest
import torch

from oracle import serving
from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _tokens(T, K, dtype, seed):
    g = gen(seed)
    x = torch.randn(T, K, generator=g) * torch.exp(torch.randn(K, generator=g))
    return x.to(dtype)


def _weights(N, K, seed):
    g = gen(seed)
    codes = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    return codes, torch.rand(N, generator=g) * 1e-2 + 1e-4, torch.randn(N, generator=g)


def _check(y, codes, scale, zero, w, wscale, bias, dtype):
    ref, size = serving.linear(codes, scale, zero, w, wscale, bias)
    err = (y.cpu().double() - ref).abs()
    bound = serving.linear_bound(dtype, ref, size)
    assert y.dtype is dtype
    assert bool((err <= bound).all()), (float((err - bound).max()), tuple(y.shape))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (5, 16), (2, 2048), (7, 2049), (4, 4096),
                                 (3, 14336), (2, 28672), (1, 65536), (33, 130)])
def test_token_codes_are_the_grids(dev, T, K, sym, dtype):
    from g2ptq_amd import quantize_tokens
    x = _tokens(T, K, dtype, 10 + T + K)
    codes, scale, zero = quantize_tokens(x.to(dev), sym=sym)
    rc, rs, rz = serving.quantize(x, 8, sym)
    assert codes.dtype is torch.int8 and codes.shape == x.shape
    assert_bitexact(scale, rs, "scale")
    assert_bitexact(codes.float(), rc, "codes")
    if sym:
        assert zero is None
    else:
        assert_bitexact(zero, rz, "zero")


@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_at_the_edges_of_the_grid(dev, sym, dtype):
    """Zero rows, one value, rows of one sign, ties, the type's largest and smallest
    values; NaN and infinite rows stay in their rows."""
    from g2ptq_amd import quantize_tokens
    K, big, tiny = 40, torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(12, K)
    x[1, 3] = 1.0
    x[2] = torch.linspace(0.5, 9, K)
    x[3] = -torch.linspace(0.5, 9, K)
    x[4] = torch.arange(K) * 0.5 - 10      # ties of the quotient
    x[4, 0] = -127.5
    x[5] = tiny * torch.arange(K)
    x[6, ::2], x[6, 1::2] = big, -big / 2
    x[7] = torch.linspace(-1, 1, K)
    x[7, 5] = float("nan")
    x[8] = torch.linspace(-1, 1, K)
    x[8, 6] = float("inf")
    x[9] = torch.linspace(-1, 1, K)
    x[9, 6] = -float("inf")
    x[10] = -0.0
    x[11] = torch.linspace(-3, 5, K)
    x = x.to(dtype)
    codes, scale, zero = quantize_tokens(x.to(dev), sym=sym)
    rc, rs, rz = serving.quantize(x, 8, sym)
    assert_bitexact(scale, rs, "scale")
    assert_bitexact(codes.float(), rc, "codes")
    if not sym:
        assert_bitexact(zero, rz, "zero")


@pytest.mark.parametrize("sym,with_bias", [(True, False), (False, True)])
@pytest.mark.parametrize("T,N,K", [
    (1, 1, 1), (1, 33, 64), (1, 4096, 512), (2, 100, 2752), (3, 5, 17), (15, 64, 4096),
    (16, 257, 100), (17, 129, 1000), (31, 16, 14336), (33, 1000, 96), (64, 64, 64),
    (65, 1024, 272), (127, 200, 515), (128, 128, 128), (129, 511, 640), (255, 257, 1040),
    (300, 768, 2048), (513, 300, 384), (777, 1000, 333), (1025, 520, 130)])
def test_linear_matches_the_exact_product(dev, T, N, K, sym, with_bias):
    from g2ptq_amd import Int8Linear
    w, wscale, bias = _weights(N, K, T + N)
    bias = bias if with_bias else None
    lin = Int8Linear(w.to(dev), wscale.to(dev), bias=None if bias is None else bias.to(dev),
                     sym=sym)
    for dtype in DTYPES:
        x = _tokens(T, K, dtype, T + K)
        rc, rs, rz = serving.quantize(x, 8, sym)
        _check(lin(x.to(dev)), rc, rs, rz, w, wscale, bias, dtype)


@pytest.mark.parametrize("T,N,K", [
    (1, 70, 32768), (1, 70, 32769), (2, 70, 16384), (2, 70, 16400), (1, 6150, 40),
    (2, 12300, 40), (16, 12300, 100), (32, 12300, 64), (33, 8193, 96), (48, 8192, 64),
    (64, 6150, 80), (64, 8200, 48), (50, 4000, 48)])
def test_each_side_of_the_choices_by_size(dev, T, N, K):
    test_linear_matches_the_exact_product(dev, T, N, K, False, True)
    test_linear_matches_the_exact_product(dev, T, N, K, True, False)


@pytest.mark.parametrize("K", [4097, 8192, 8200, 16384, 16391])
def test_token_codes_of_long_rows(dev, K):
    for dtype in DTYPES:
        test_token_codes_are_the_grids(dev, 3, K, K % 2 == 0, dtype)


@pytest.mark.parametrize("T", [1, 16, 40, 200, 600])
def test_extreme_codes_and_zero_points(dev, T):
    """The sums' range: every code at an end of the grid, K at its limit."""
    from g2ptq_amd import Int8Linear, quantize_tokens, int8_matmul
    K, N = 65536, 24
    w = torch.full((N, K), -128, dtype=torch.int8)
    w[1::2] = 127
    x = torch.full((T, K), 3.0)   # one sign: zero point at the end, code - zero = 255
    x[1::2] = -2.0
    lin = Int8Linear(w.to(dev), torch.full((N,), 2.0 ** -10, device=dev), sym=False)
    rc, rs, rz = serving.quantize(x, 8, False)
    assert float((rc - rz[:, None]).abs().max()) == 255
    _check(lin(x.to(dev)), rc, rs, rz, w, torch.full((N,), 2.0 ** -10), None, torch.float32)
    c, s, z = quantize_tokens(x.to(dev), sym=False)
    assert_bitexact(int8_matmul(c, s, lin, zero=z, dtype=torch.float32), lin(x.to(dev)), "apart")


@pytest.mark.parametrize("T", [1, 20, 300])
def test_large_weights_stream_in_full(dev, T):
    """One whole projection of the benchmark's hidden size."""
    from g2ptq_amd import Int8Linear
    N, K = 4096, 4096
    w, wscale, _ = _weights(N, K, 5)
    x = _tokens(T, K, torch.bfloat16, 6)
    y = Int8Linear(w.to(dev), wscale.to(dev))(x.to(dev))
    rc, rs, rz = serving.quantize(x, 8, True)
    _check(y, rc, rs, rz, w, wscale, None, torch.bfloat16)


def test_strides_shapes_and_alignment(dev):
    from g2ptq_amd import Int8Linear
    K, N = 200, 48
    w, wscale, bias = _weights(N, K, 1)
    lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev))
    base = _tokens(64, 3 * K + 5, torch.bfloat16, 2).to(dev)
    for x in (base[:, 1:1 + K], base[:, 8:8 + K], base[::3, 3:3 + K], base[:4, :K].flip(0),
              base.t()[:K, :9].t(), base[:1, 5:5 + K].expand(6, K),
              base[:60, :K].unflatten(0, (5, 12)), base[0, :K], base[:0, :K]):
        y = lin(x)
        assert y.shape == x.shape[:-1] + (N,)
        ref = lin(x.reshape(-1, K).clone())
        assert_bitexact(y.reshape(-1, N), ref, str(x.shape))


def test_shared_tokens_give_what_the_linear_gives(dev):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    x = _tokens(70, 333, torch.float16, 3).to(dev).unflatten(0, (7, 10))
    for sym in (True, False):
        codes, scale, zero = quantize_tokens(x, sym=sym)
        assert codes.shape == x.shape and scale.shape == x.shape[:-1]
        for N in (64, 31):
            w, wscale, bias = _weights(N, 333, N)
            lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=sym)
            y = int8_matmul(codes, scale, lin, zero=zero, dtype=torch.float16)
            assert_bitexact(y, lin(x), "padded view")
            own = codes.contiguous()  # odd row stride: laid out again
            assert_bitexact(int8_matmul(own, scale, lin, zero=zero, dtype=torch.float16), y, "own")


@pytest.mark.parametrize("T", [1, 40, 300])
def test_bad_rows_stay_in_their_rows(dev, T):
    from g2ptq_amd import Int8Linear
    w, wscale, _ = _weights(100, 160, 4)
    lin = Int8Linear(w.to(dev), wscale.to(dev))
    x = _tokens(T, 160, torch.bfloat16, 4).to(dev)
    good = lin(x)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[T // 2, 7] = bad
        got = lin(y)
        assert bool(got[T // 2].isnan().all())
        keep = torch.arange(T) != T // 2
        assert_bitexact(got[keep.to(dev)], good[keep.to(dev)], str(bad))
    zero = torch.zeros_like(x)
    assert float(lin(zero).abs().max()) == 0.0


def test_another_stream_and_a_graph(dev):
    from g2ptq_amd import Int8Linear
    w, wscale, _ = _weights(512, 1024, 7)
    lin = Int8Linear(w.to(dev), wscale.to(dev))
    for T in (1, 24, 400):
        x = _tokens(T, 1024, torch.bfloat16, T).to(dev)
        ref = lin(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = lin(x)
        torch.cuda.current_stream().wait_stream(side)
        assert_bitexact(y, ref, f"stream T={T}")
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(static)
        for k in range(3):
            static.copy_(_tokens(T, 1024, torch.bfloat16, 50 + k).to(dev))
            graph.replay()
            torch.cuda.synchronize()
            assert_bitexact(out, lin(static), f"replay {k} T={T}")


def test_from_export_and_from_linear(dev):
    """An 8-bit per-channel GPTQ export, and round-to-nearest, run as linears."""
    from g2ptq_amd import GPTQ, Int8Linear, WeightQuantizer, make_group_quantizers
    g = gen(11)
    R, C = 96, 130
    lin = torch.nn.Linear(C, R, bias=True)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(R, C, generator=g) * 0.02)
        lin.bias.copy_(torch.randn(R, generator=g))
    lin = lin.to(dev)
    x = _tokens(512, C, torch.float32, 12).to(dev)
    gq = GPTQ([lin])
    q = WeightQuantizer()
    q.configure(8, perchannel=True, sym=True)
    gq.quantizer = make_group_quantizers(q, C, -1)
    gq.add_batch(0, x.reshape(1, 512, C), None)
    gq.fasterquant(blocksize=128, percdamp=0.01, groupsize=-1, backend="hip",
                   export_compressed_tensors=True)
    run = Int8Linear.from_export(lin)
    assert_bitexact(run.weight[:, :C].float() * run.weight_scale[:, None], lin.weight, "export")
    rc, rs, rz = serving.quantize(x.cpu(), 8, True)
    _check(run(x), rc, rs, rz, run.weight[:, :C].cpu(), run.weight_scale.cpu(), lin.bias.cpu(),
           torch.float32)
    q = WeightQuantizer()
    q.configure(8, perchannel=True, sym=True)
    q.find_params(lin.weight.data)
    rtn = Int8Linear.from_linear(lin, q)
    dq, _, _ = q.fake_quantize(lin.weight.data)
    assert_bitexact(rtn.weight[:, :C].float() * rtn.weight_scale[:, None], dq, "rtn")
    with pytest.raises(ValueError, match="one group per row"):
        Int8Linear.from_export({"weight_packed": torch.zeros(4, 2, dtype=torch.int32, device=dev),
                                "weight_scale": torch.ones(4, 2, device=dev),
                                "weight_shape": torch.tensor([4, 8])})
    with pytest.raises(ValueError, match="no 8-bit codes"):
        Int8Linear.from_export({"weight_packed": torch.zeros(4, 1, dtype=torch.int32, device=dev),
                                "weight_scale": torch.ones(4, 1, device=dev),
                                "weight_shape": torch.tensor([4, 8])})


def test_refusals(dev):
    from g2ptq_amd import Int8Linear, _lib, int8_matmul, quantize_tokens
    w, wscale, _ = _weights(8, 32, 1)
    lin = Int8Linear(w.to(dev), wscale.to(dev))
    x = torch.zeros(4, 32, device=dev)
    with pytest.raises(NotImplementedError):
        lin(x.double())
    with pytest.raises(ValueError, match="last dimension"):
        lin(x[:, :31])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lin(x.cpu())
    with pytest.raises(RuntimeError, match="inference only"):
        lin(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="one scale"):
        Int8Linear(w.to(dev), wscale[:5].to(dev))
    with pytest.raises(ValueError, match="columns"):
        Int8Linear(torch.zeros(1, 65537, dtype=torch.int8, device=dev), torch.ones(1, device=dev))
    with pytest.raises(ValueError, match="rows of 1"):
        quantize_tokens(torch.zeros(1, 65537, device=dev))
    codes, scale, zero = quantize_tokens(x, sym=False)
    with pytest.raises(ValueError, match="sym=False"):
        int8_matmul(codes, scale, lin, zero=zero)
    with pytest.raises(ValueError, match="scale"):
        int8_matmul(codes, scale[:2], lin)
    p = _lib.ptr
    y = torch.empty(6, 8, device=dev)
    wide = torch.zeros(6, 32, dtype=torch.int8, device=dev)
    x, scale = torch.zeros(6, 32, device=dev), torch.zeros(6, device=dev)
    ldw = lin.weight.stride(0)
    for ldc, ldb in ((24, ldw), (32, 48)):
        with pytest.raises(ValueError, match="16-byte aligned rows"):
            _lib.call("g2ptq_int8_gemm", _lib.stream_ptr(), p(wide), ldc, p(scale), None,
                      p(lin.weight), ldb, p(lin.weight_scale), None, None, 6, 8, 32, p(y), 2, 8,
                      None, 0)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("g2ptq_int8_linear", _lib.stream_ptr(), p(x), 2, 6, 32, 32, 1, p(lin.weight),
                  ldw, p(lin.weight_scale), None, None, 8, p(y), 8, None, 0)
