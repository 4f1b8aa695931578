"""GPU: norms with the residual's addition and their 8-bit codes, and rotary positions, against
the definitions in 64 bits: types, ragged and strided rows, extreme values, long positions."""
import math

import pytest
import torch

from oracle import layer_ops, serving
from tests._util import assert_bitexact, gen

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _x(*shape, dtype, seed):
    g = gen(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(0.7 * torch.randn(shape[-1], generator=g))
    return (x * torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)


def _check_norm(y, x, w, eps, dtype, residual=None, total=None):
    ref, s = layer_ops.rms_norm(x, w, eps, residual)
    bound = layer_ops.rounded(dtype, ref, layer_ops.rms_norm_error(x.shape[-1]) * ref.abs())
    assert y.dtype is dtype and y.shape == x.shape and y.is_contiguous()
    err = (y.cpu().double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())
    if total is not None:
        bound = layer_ops.rounded(dtype, s, layer_ops.E * s.abs())
        assert total.dtype is dtype and bool(((total.cpu().double() - s).abs() <= bound).all())


SIZES = [(1, 1), (3, 7), (5, 16), (300, 64), (33, 65), (7, 96), (1000, 128), (9, 129), (17, 256),
         (5, 300), (6, 512), (3, 520), (5, 1000), (4, 1024), (3, 1030), (2, 2048), (3, 2050),
         (2, 2752), (5, 4096), (2, 4100), (3, 8192), (2, 8200), (2, 16384), (2, 16390), (1, 65536)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,C", SIZES)
def test_norm_is_the_formula(dev, T, C, dtype):
    from g2ptq_amd import rms_norm
    x, r = _x(T, C, dtype=dtype, seed=T + C), _x(T, C, dtype=dtype, seed=T + C + 1)
    for i, wtype in enumerate(DTYPES):
        w = (1 + 0.5 * torch.randn(C, generator=gen(C))).to(wtype)
        eps = (1e-5, 0.1, 1e-6)[i]
        _check_norm(rms_norm(x.to(dev), w.to(dev), eps), x, w, eps, dtype)
        y, s = rms_norm(x.to(dev), w.to(dev), eps, residual=r.to(dev))
        _check_norm(y, x, w, eps, dtype, r, s)


@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("T,C", SIZES)
def test_codes_are_the_grids(dev, T, C, sym):
    """In fp32 the values are what is quantized; bf16 and fp16 inputs go the same way."""
    from g2ptq_amd import rms_norm_quantize
    w = (1 + 0.5 * torch.randn(C, generator=gen(C))).to(dev)
    for dtype in DTYPES:
        x = _x(T, C, dtype=dtype, seed=T + C).to(dev)
        r = _x(T, C, dtype=dtype, seed=T + C + 1).to(dev)
        for res in (None, r):
            wide = rms_norm_quantize(x.float(), w, 1e-5, sym=sym, values=True,
                                     residual=None if res is None else res.float())
            _check_norm(wide.values, x.float().cpu(), w.cpu(), 1e-5, torch.float32,
                        None if res is None else res.float().cpu(), wide.sum)
            rc, rs, rz = serving.quantize(wide.values.cpu(), 8, sym)
            got = rms_norm_quantize(x, w, 1e-5, residual=res, sym=sym, values=dtype != torch.float16)
            for t in (wide, got):
                assert t.codes.dtype is torch.int8 and t.codes.shape == x.shape
                assert_bitexact(t.codes.float(), rc, "codes")
                assert_bitexact(t.scale, rs, "scale")
                assert (t.zero is None) == sym
                if not sym:
                    assert_bitexact(t.zero, rz, "zero")
            assert (got.sum is None) == (res is None)
            assert (got.values is None) == (dtype is torch.float16)
            if got.values is not None:
                assert_bitexact(got.values, wide.values.to(dtype), "values")
            if res is not None:
                assert_bitexact(got.sum, wide.sum.to(dtype), "sum")


@pytest.mark.parametrize("C", [8193, 16384])
def test_many_long_rows(dev, C):
    from g2ptq_amd import rms_norm, rms_norm_quantize
    w = (1 + 0.5 * torch.randn(C, generator=gen(C))).to(dev)
    for dtype in (torch.bfloat16, torch.float32):
        for T in (512, 513):
            x = _x(T, C, dtype=dtype, seed=T).to(dev)
            r = _x(T, C, dtype=dtype, seed=T + 1).to(dev)
            y, s = rms_norm(x, w, 1e-5, residual=r)
            _check_norm(y, x.cpu(), w.cpu(), 1e-5, dtype, r.cpu(), s)
            q = rms_norm_quantize(x, w, 1e-5, residual=r)
            for part in (slice(0, 3), slice(T - 3, T)):
                p = rms_norm_quantize(x[part], w, 1e-5, residual=r[part])
                assert_bitexact(q.codes[part], p.codes, "codes")
                assert_bitexact(q.scale[part], p.scale, "scale")


def test_strided_rows(dev):
    """Heads of a projection, columns of a wider matrix, transposed and expanded leading
    dimensions, single rows, rows off 16 bytes; residuals laid out otherwise than their rows."""
    from g2ptq_amd import rms_norm, rms_norm_quantize
    for dtype in DTYPES:
        big = _x(6, 5, 4, 72, dtype=dtype, seed=3).to(dev)
        views = [big[:, :, 1:3], big[:, 2], big[..., 8:], big[..., 3:40], big[::2, :, :, :64],
                 big.transpose(0, 2), big[1:2, :, 3:4], big[0, 0, 0], big[:, :, :1].expand(6, 5, 9, 72),
                 big.permute(3, 0, 1, 2)[::2], big[:0], big.transpose(1, 3)]
        for v in views:
            w = (1 + 0.1 * torch.randn(v.shape[-1], generator=gen(1))).to(dev)
            ref = rms_norm(v.contiguous(), w)
            assert_bitexact(rms_norm(v, w), ref, str(v.stride()))
            wide = torch.zeros(*v.shape[:-1], v.shape[-1] + 8, dtype=dtype, device=dev)
            for r in (v.contiguous(), wide[..., 8:], v):
                y, s = rms_norm(v, w, residual=r)
                y2, s2 = rms_norm(v.contiguous(), w, residual=r.contiguous())
                assert_bitexact(y, y2, "y")
                assert_bitexact(s, s2, "s")
            t, t2 = rms_norm_quantize(v, w), rms_norm_quantize(v.contiguous(), w)
            assert t.codes.shape == v.shape and t.scale.shape == v.shape[:-1]
            assert_bitexact(t.codes, t2.codes, "codes")
            assert_bitexact(t.scale, t2.scale, "scale")


@pytest.mark.parametrize("C", [1, 7, 9, 15, 63, 333, 2051, 4097, 9001])
def test_rows_beside_nan(dev, C):
    """Rows at any address of their type with NaN on every side, which no row takes in."""
    from g2ptq_amd import rms_norm, rms_norm_quantize
    for dtype in DTYPES:
        x, r = _x(6, C, dtype=dtype, seed=C).to(dev), _x(6, C, dtype=dtype, seed=C + 1).to(dev)
        w = (1 + 0.1 * torch.randn(C, generator=gen(2))).to(dev, dtype)
        y, s = rms_norm(x, w, residual=r)
        q = rms_norm_quantize(x, w, residual=r)
        assert not y.isnan().any()
        for before, behind in ((1, 0), (2, 1), (5, 3), (8, 8)):
            def inside(v):
                wide = torch.full((*v.shape[:-1], before + C + behind), float("nan"), dtype=dtype,
                                  device=dev)
                wide[..., before:before + C] = v
                return wide[..., before:before + C]

            got = rms_norm(inside(x), inside(w), residual=inside(r))
            assert_bitexact(got[0], y, f"{before} {behind}")
            assert_bitexact(got[1], s, f"{before} {behind} sum")
            got = rms_norm_quantize(inside(x), inside(w), residual=inside(r))
            assert_bitexact(got.codes, q.codes, f"{before} {behind} codes")
            assert_bitexact(got.scale, q.scale, f"{before} {behind} scale")
            assert_bitexact(got.sum, q.sum, f"{before} {behind} sum")


@pytest.mark.parametrize("C", [40, 500, 2000, 5000, 20000])
def test_rows_of_extreme_values(dev, C):
    """Squares that overflow or vanish in fp32, rows of zeros, NaN and infinities; their rows
    only."""
    from g2ptq_amd import rms_norm, rms_norm_quantize
    base = _x(12, C, dtype=torch.float32, seed=1)
    x = base.clone()
    x[1] *= 1e25
    x[2] *= 1e-25
    x[3] = 0
    x[4, 3] = float("nan")
    x[5, 7] = float("inf")
    x[6, 9] = -float("inf")
    x[7] = 3e38
    x[8] *= 1e-42
    x[9] = 0
    x[9, 11] = 1e-30
    w = torch.ones(C)
    for eps in (1e-6, 1e-30, 0.0, 1e30):
        y = rms_norm(x.to(dev), w.to(dev), eps).cpu()
        s = rms_norm_quantize(x.to(dev), w.to(dev), eps, values=True)
        ref, _ = layer_ops.rms_norm(x, w, eps)
        for i in range(12):
            zero = i == 3 and eps == 0
            assert bool(y[i].isnan().all()) == (zero or i == 4), i
            if i in (5, 6):
                at = x[i].isinf()
                assert bool(y[i][at].isnan().all()) and bool((y[i][~at] == 0).all())
            if i in (4, 5, 6) or zero:
                assert bool(s.scale[i].isnan()) and bool((s.codes[i] == 0).all())
                continue
            # (values below fp32's normal range keep half a unit of 2^-149)
            bound = layer_ops.rms_norm_error(C) * ref[i].abs() + 2.0 ** -149
            if i == 8 and eps == 1e30:
                bound = bound + 2.0 ** -149
            assert bool(((y[i].double() - ref[i]).abs() <= bound).all()), (i, eps)
            assert_bitexact(s.values[i], y[i], "values")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,C", [(3, 100), (5, 1000), (3, 4096), (3, 8192), (512, 8200), (513, 8200),
                                 (2, 16384), (3, 16390), (513, 16384)])
def test_sum_and_values_in_place(dev, T, C, dtype):
    """A caller of the C entry updates its residual's stream in place: the sum over either
    addend, the values over the other, on both sides of the rule for long rows."""
    from g2ptq_amd import _lib
    from g2ptq_amd.norm_utils import _DTYPE_CODE
    code, ldc = _DTYPE_CODE[dtype], -(-C // 64) * 64
    w = (1 + 0.5 * torch.randn(C, generator=gen(C))).to(dev)
    x0 = torch.randn(T, C, generator=gen(T), dtype=torch.float32).to(dtype).to(dev)
    r0 = torch.randn(T, C, generator=gen(C), dtype=torch.float32).to(dtype).to(dev)

    def run(x, r, y, total, quantize, sym):
        codes = torch.zeros(T, ldc, dtype=torch.int8, device=dev)
        scale, zero = torch.zeros(2, T, device=dev).unbind()
        _lib.call("g2ptq_rms_norm", _lib.current_stream(), x.data_ptr(), C, 0, r.data_ptr(), C, 0,
                  code, w.data_ptr(), 2, T, 1, C, 1e-6, y.data_ptr(), total.data_ptr(), sym,
                  codes.data_ptr() if quantize else None, ldc, scale.data_ptr(), zero.data_ptr())
        return y, total, codes, scale, zero

    for quantize, sym in ((False, 1), (True, 1), (True, 0)):
        want = run(x0, r0, torch.empty_like(x0), torch.empty_like(x0), quantize, sym)
        for sum_at, y_at in ((0, None), (1, None), (None, 0), (None, 1), (0, 1), (1, 0)):
            pair = [x0.clone(), r0.clone()]
            y, total = (torch.empty_like(x0) if at is None else pair[at] for at in (y_at, sum_at))
            got = run(*pair, y, total, quantize, sym)
            for name, a, b in zip(("values", "sum", "codes", "scale", "zero"), got, want):
                assert_bitexact(a, b, f"{name}, sum over {sum_at}, values over {y_at}")


def test_dequantized_tokens_are_what_codes_stand_for(dev):
    from g2ptq_amd import dequantize_tokens, quantize_tokens
    for T, K in ((1, 1), (3, 7), (40, 130), (5, 16), (2, 4096), (700, 2752), (1, 65536)):
        for sym in (True, False):
            x = _x(T, K, dtype=torch.float32, seed=K)
            x[0] = 0
            c, s, z = quantize_tokens(x.to(dev), sym=sym)
            exact = serving.dequantize(c.cpu(), s.cpu(), torch.zeros(T) if sym else z.cpu())
            for dtype in DTYPES:
                for codes in (c, c.contiguous(), c.t().contiguous().t()):
                    y = dequantize_tokens(codes, s, z, dtype=dtype)
                    assert y.dtype is dtype and y.shape == x.shape
                    if dtype is torch.float32:
                        assert_bitexact(y, exact.float(), "values")
                    # (the product is rounded to the type, by way of fp32 or, where the hardware
                    # has one instruction for both, at once)
                    bound = layer_ops.rounded(dtype, exact, layer_ops.E * exact.abs())
                    assert bool(((y.cpu().double() - exact).abs() <= bound).all())
    c, s, _ = quantize_tokens(_x(2, 3, 37, dtype=torch.float16, seed=1).to(dev))
    assert dequantize_tokens(c, s).shape == (2, 3, 37)
    assert dequantize_tokens(c[0, 0], s[0, 0]).shape == (37,)
    assert dequantize_tokens(c[:0], s[:0]).shape == (0, 3, 37)
    s[0, 1] = float("nan")
    assert bool(dequantize_tokens(c, s)[0, 1].isnan().all())


def test_norm_feeds_the_products(dev):
    from g2ptq_amd import Int8Linear, int8_matmul, rms_norm_quantize
    g = gen(4)
    lin = Int8Linear(torch.randint(-128, 128, (70, 130), generator=g, dtype=torch.int8).to(dev),
                     torch.rand(70, generator=g).to(dev), sym=False)
    x, w = _x(33, 130, dtype=torch.float16, seed=2).to(dev), torch.ones(130, device=dev)
    t = rms_norm_quantize(x.float(), w, sym=False, values=True)
    assert_bitexact(int8_matmul(t.codes, t.scale, lin, zero=t.zero, dtype=torch.float32),
                    lin(t.values), "product")


def test_norm_refusals(dev):
    from g2ptq_amd import dequantize_tokens, rms_norm, rms_norm_quantize
    x, w = torch.ones(3, 8, device=dev), torch.ones(8, device=dev)
    for f in (rms_norm, rms_norm_quantize):
        for err, call in (
                (NotImplementedError, lambda: f(x.double(), w)), (ValueError, lambda: f(x, w[:7])),
                (ValueError, lambda: f(x, w.double())), (ValueError, lambda: f(x, w, -1.0)),
                (ValueError, lambda: f(x, w, float("nan"))), (RuntimeError, lambda: f(x.cpu(), w)),
                (ValueError, lambda: f(x[0, 0], w[0])),
                (RuntimeError, lambda: f(x, w.cpu())), (ValueError, lambda: f(x[:, :0], w[:0])),
                (ValueError, lambda: f(x, w, residual=x[:2])),
                (ValueError, lambda: f(x, w, residual=x.half())),
                (RuntimeError, lambda: f(x, w, residual=x.cpu())),
                (RuntimeError, lambda: f(x.clone().requires_grad_(), w)),
                (RuntimeError, lambda: f(x, w.clone().requires_grad_())),
                (RuntimeError, lambda: f(x, w, residual=x.clone().requires_grad_())),
                (ValueError, lambda: f(torch.ones(1, 65537, device=dev),
                                       torch.ones(65537, device=dev)))):
            with pytest.raises(err):
                call()
    c, s = torch.zeros(3, 8, dtype=torch.int8, device=dev), torch.ones(3, device=dev)
    for err, call in ((ValueError, lambda: dequantize_tokens(x, s)),
                      (ValueError, lambda: dequantize_tokens(c, s[:2])),
                      (ValueError, lambda: dequantize_tokens(c, s, s.double())),
                      (ValueError, lambda: dequantize_tokens(c, s.cpu())),
                      (RuntimeError, lambda: dequantize_tokens(c.cpu(), s.cpu())),
                      (NotImplementedError, lambda: dequantize_tokens(c, s, dtype=torch.int8))):
        with pytest.raises(err):
            call()


def test_rows_past_32_bits(dev):
    """Values beyond the 2^32nd, and more rows than one launch takes."""
    from g2ptq_amd import rms_norm
    x = torch.zeros((1 << 26) + 3, 72, dtype=torch.bfloat16, device=dev)
    tail = _x(3, 72, dtype=torch.bfloat16, seed=1)
    x[-3:] = tail.to(dev)
    w = torch.ones(72, device=dev)
    y = rms_norm(x, w)
    _check_norm(y[-3:], tail, w.cpu(), 1e-6, torch.bfloat16)
    assert not bool(y[:1000].any()) and not bool(y[-1000:-3].any())
    del x, y
    x = torch.zeros((1 << 23) + 2, 1, dtype=torch.bfloat16, device=dev).expand(-1, 1032)
    x = torch.cat([x[:1], x[:1] + 2]).repeat_interleave(torch.tensor([1 << 23, 2], device=dev), 0)
    y = rms_norm(x, torch.ones(1032, device=dev))
    assert not bool(y[:1 << 23].any()) and bool((y[1 << 23:] == 1).all())
    del x, y
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------

SCALINGS = [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 16.0, "original_positions": 4096},
            {"type": "yarn", "factor": 4.0, "original_positions": 2048, "beta_fast": 16,
             "beta_slow": 2, "attention_factor": 0.75},
            {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_positions": 8192}]


def _positions(T, seed):
    p = torch.randint(0, 200000, (T,), generator=gen(seed))
    p[::3] = torch.arange(len(p[::3]))
    if T > 4:
        p[1], p[2], p[4] = 2 ** 31 + 12345, -17, 2 ** 40 + 1
    return p


def _check_rotary(rotary, got, x, positions):
    assert got.dtype is x.dtype and got.shape == x.shape and got.is_contiguous()
    ref, err = layer_ops.rotary(x, positions, rotary.frequencies, rotary.factor,
                                rotary.rotary_dim, rotary.layout == "interleaved")
    bound = layer_ops.rounded(x.dtype, ref, err)
    off = (got.cpu().double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
    # channels that stay keep their bits
    assert_bitexact(got[..., rotary.rotary_dim:], x[..., rotary.rotary_dim:], "rest")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,part", [(2, 2), (16, 2), (64, 64), (64, 32), (80, 80), (80, 20),
                                      (96, 96), (128, 128), (128, 6), (192, 64), (250, 250),
                                      (255, 130), (256, 256), (1024, 1024)])
def test_rotary_is_the_formula(dev, dim, part, layout):
    from g2ptq_amd import Rotary
    for i, dtype in enumerate(DTYPES):
        rotary = Rotary(dim, rotary_dim=part, base=(10000.0, 500000.0, 100.0)[i], layout=layout)
        for T, H, K in ((1, 1, 1), (1, 32, 8), (7, 3, 1), (70, 4, 2)):
            q, k = _x(T, H, dim, dtype=dtype, seed=T), _x(T, K, dim, dtype=dtype, seed=T + 1)
            p = _positions(T, T)
            a, b = rotary(q.to(dev), k.to(dev), p.to(dev))
            _check_rotary(rotary, a, q, p)
            _check_rotary(rotary, b, k, p)


@pytest.mark.parametrize("scaling", SCALINGS, ids=str)
def test_rotary_frequencies_are_the_formulas(dev, scaling):
    from g2ptq_amd import Rotary, rotary_frequencies
    d, base = 128, 10000.0
    theta, m = rotary_frequencies(d, base, scaling)
    kind, s = (scaling["type"], scaling["factor"]) if scaling else (None, 1.0)
    for i in range(d // 2):
        f = base ** (-2 * i / d)
        want, factor = f, 1.0
        if kind == "linear":
            want = f / s
        elif kind == "ntk":
            want = (base * s ** (d / (d - 2))) ** (-2 * i / d)
        elif kind == "yarn":
            L = scaling["original_positions"]
            fast, slow = scaling.get("beta_fast", 32), scaling.get("beta_slow", 1)
            lo = math.floor(d / 2 * math.log(L / (2 * math.pi * fast)) / math.log(base))
            hi = math.ceil(d / 2 * math.log(L / (2 * math.pi * slow)) / math.log(base))
            mix = min(1.0, max(0.0, (i - lo) / (hi - lo)))
            want = f / s * mix + f * (1 - mix)
            factor = scaling.get("attention_factor", 1 + 0.1 * math.log(s))
        elif kind == "bands":
            turns = scaling["original_positions"] * f / (2 * math.pi)
            want = f if turns > 4 else f / s if turns < 1 else \
                (turns - 1) / 3 * f + (4 - turns) / 3 * f / s
        assert math.isclose(float(theta[i]), want, rel_tol=1e-12)
        assert math.isclose(m, factor, rel_tol=1e-12)
    rotary = Rotary(d, scaling=scaling)
    q, p = _x(40, 2, d, dtype=torch.float32, seed=1), _positions(40, 2)
    out, none = rotary(q.to(dev), None, p.to(dev))
    assert none is None
    _check_rotary(rotary, out, q, p)
    given = Rotary(d, frequencies=theta, attention_factor=m)
    assert_bitexact(given(q.to(dev), None, p.to(dev))[0], out, "given frequencies")
    given = Rotary(d, frequencies=theta.tolist(), attention_factor=m)
    assert_bitexact(given(q.to(dev), None, p.to(dev))[0], out, "given numbers")


def test_rotary_strides(dev):
    """Views of a projection's output, transposed layouts, rows off 16 bytes, expanded heads;
    no tokens and no heads."""
    from g2ptq_amd import Rotary
    for dtype in (torch.bfloat16, torch.float32):
        for layout in ("half", "interleaved"):
            rotary = Rotary(64, rotary_dim=48, layout=layout)
            qkv = _x(9, 8, 64, dtype=dtype, seed=1).to(dev)
            odd = _x(9, 8, 69, dtype=dtype, seed=2).to(dev)[..., 3:67]
            p = _positions(9, 3).to(dev)
            for q, k in ((qkv[:, :5], qkv[:, 5:7]), (odd, qkv[:, ::3]),
                         (qkv.transpose(0, 1).contiguous().transpose(0, 1), odd[:, 1:2]),
                         (qkv[:, :1].expand(9, 6, 64), odd),
                         (qkv.transpose(1, 2).contiguous().transpose(1, 2), qkv[:, :0])):
                a, b = rotary(q, k, p)
                c, d = rotary(q.contiguous(), k.contiguous(), p.clone())
                assert_bitexact(a, c, "q")
                assert_bitexact(b, d, "k")
                _check_rotary(rotary, a, q.cpu(), p.cpu())
            wide = torch.stack([p, p], 1)[:, 0]
            assert_bitexact(rotary(qkv, qkv, wide)[1], rotary(qkv, qkv, p)[0], "positions")
            assert rotary(qkv[:0], qkv[:0, :2], p[:0])[1].shape == (0, 2, 64)


@pytest.mark.parametrize("dim,part", [(2, 2), (10, 6), (18, 18), (36, 14), (70, 70), (134, 66)])
def test_rotary_heads_beside_nan(dev, dim, part):
    """Heads at any address of their type with NaN on every side."""
    from g2ptq_amd import Rotary
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for layout in ("half", "interleaved"):
            rotary = Rotary(dim, rotary_dim=part, layout=layout)
            q, k = (_x(9, h, dim, dtype=dtype, seed=h).to(dev) for h in (5, 2))
            p = _positions(9, 3).to(dev)
            a, b = rotary(q, k, p)
            assert not a.isnan().any() and not b.isnan().any()
            for before, behind in ((1, 0), (3, 2), (8, 8)):
                def inside(v):
                    wide = torch.full((*v.shape[:-1], before + dim + behind), float("nan"),
                                      dtype=dtype, device=dev)
                    wide[..., before:before + dim] = v
                    return wide[..., before:before + dim]

                got = rotary(inside(q), inside(k), p)
                assert_bitexact(got[0], a, f"{before} {behind} q")
                assert_bitexact(got[1], b, f"{before} {behind} k")


def test_rotary_turns_back(dev):
    """Negative positions are the inverse."""
    from g2ptq_amd import Rotary
    rotary = Rotary(64, layout="interleaved")
    q, p = _x(20, 2, 64, dtype=torch.float32, seed=1).to(dev), _positions(20, 2).to(dev)
    back, _ = rotary(rotary(q, None, p)[0], None, -p)
    torch.testing.assert_close(back, q, rtol=0, atol=2.0 ** -20 * float(q.abs().max()))


def test_rotary_keeps_nan_and_infinities_in_their_pairs(dev):
    from g2ptq_amd import Rotary
    q = _x(3, 2, 64, dtype=torch.bfloat16, seed=1)
    clean = Rotary(64)(q.to(dev), None, torch.arange(3, device=dev))[0]
    q[1, 0, 5], q[2, 1, 40] = float("nan"), float("inf")
    out = Rotary(64)(q.to(dev), None, torch.arange(3, device=dev))[0].cpu()
    bad = torch.zeros(3, 2, 64, dtype=torch.bool)
    bad[1, 0, 5] = bad[1, 0, 37] = bad[2, 1, 8] = bad[2, 1, 40] = True
    assert not bool(out[bad].isfinite().any())
    assert_bitexact(out[~bad], clean.cpu()[~bad], "others")


def test_rotary_refusals(dev):
    from g2ptq_amd import Rotary, rotary_frequencies
    for kw in ({"rotary_dim": 3}, {"rotary_dim": 66}, {"rotary_dim": 0}, {"layout": "pairs"},
               {"scaling": {"type": "magic", "factor": 2}}, {"scaling": {"type": "linear"}},
               {"scaling": {"type": "linear", "factor": 0}}, {"base": 0.0},
               {"scaling": {"type": "yarn", "factor": 2}}, {"frequencies": torch.ones(5)},
               {"scaling": {"type": "linear", "factor": 2, "more": 1}}):
        with pytest.raises(ValueError):
            Rotary(64, **kw)
    with pytest.raises(ValueError):
        Rotary(1026)
    with pytest.raises(RuntimeError):
        Rotary(64, device="cpu")
    with pytest.raises(ValueError):
        rotary_frequencies(7)
    r = Rotary(64)
    q, p = torch.ones(3, 2, 64, device=dev), torch.arange(3, device=dev)
    for err, call in ((ValueError, lambda: r(q, q, p[:2])), (ValueError, lambda: r(q, q[:2], p)),
                      (ValueError, lambda: r(q[..., :32], q, p)), (ValueError, lambda: r(q, q, p.int())),
                      (ValueError, lambda: r(q, q, p.cpu())), (ValueError, lambda: r(q[0], q, p)),
                      (ValueError, lambda: r(q, q, p[0])),
                      (NotImplementedError, lambda: r(q, q.half(), p)),
                      (NotImplementedError, lambda: r(q.double(), q.double(), p)),
                      (RuntimeError, lambda: r(q.cpu(), q, p)),
                      (RuntimeError, lambda: r(q, q.clone().requires_grad_(), p))):
        with pytest.raises(err):
            call()


def test_rotary_past_32_bits(dev):
    """Elements beyond the 2^32nd: the last token like the first."""
    from g2ptq_amd import Rotary
    T = (1 << 25) + 5
    rotary = Rotary(64)
    q = torch.zeros(T, 2, 64, dtype=torch.bfloat16, device=dev)
    row = _x(1, 2, 64, dtype=torch.bfloat16, seed=1)
    q[-1] = row[0].to(dev)
    p = torch.arange(T, device=dev)
    out, _ = rotary(q, None, p)
    _check_rotary(rotary, out[-1:], row, p[-1:].cpu())
    assert not bool(out[:1000].any()) and not bool(out[-1000:-1].any())
    del q, out
    torch.cuda.empty_cache()


def test_rotary_past_the_first_launch(dev):
    """One token a workgroup and more tokens than a launch has: the last ones lie in the second."""
    from g2ptq_amd import Rotary
    T, H = (1 << 23) + 3, 160
    for layout in ("half", "interleaved"):
        rotary = Rotary(2, layout=layout)
        q = _x(3, H, 2, dtype=torch.bfloat16, seed=7)
        k = _x(3, 1, 2, dtype=torch.bfloat16, seed=8)
        # (inputs of one token for all but the last three; an output of 5 GB)
        p = torch.zeros(T, dtype=torch.int64, device=dev)
        p[-3:] = torch.tensor([5, 1 << 33, -7], device=dev)
        wide = torch.zeros(T, 1, 2, dtype=torch.bfloat16, device=dev)
        wide[-3:] = k.to(dev)
        out, kout = rotary(wide.expand(T, H, 2), wide, p)
        _check_rotary(rotary, out[-3:], k.expand(3, H, 2), p[-3:].cpu())
        _check_rotary(rotary, kout[-3:], k, p[-3:].cpu())
        assert not bool(out[-1000:-3].any()) and not bool(out[:1000].any())
        assert not bool(kout[:-3].any())
        del out, kout
        torch.cuda.empty_cache()
        got, _ = rotary(q.to(dev), None, p[-3:])
        _check_rotary(rotary, got, q, p[-3:].cpu())


@pytest.mark.parametrize("what", ["rms_norm", "rms_norm_quantize", "dequantize_tokens", "rotary",
                                  "adapters"])
def test_tangents_are_refused(dev, what):
    """A tangent raises, in every argument that may carry one, and the primal alone is served."""
    from torch.autograd import forward_ad

    from g2ptq_amd import LowRankAdapters, Rotary, dequantize_tokens, rms_norm, rms_norm_quantize
    x = torch.randn(3, 64, generator=gen(1)).to(dev)
    w, codes = torch.ones(64, device=dev), torch.ones(3, 64, dtype=torch.int8, device=dev)
    p, index = torch.arange(3, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    half = x.half()
    set_ = LowRankAdapters([half[:2].contiguous()], [half[:, :2].contiguous()])
    rotary = Rotary(64)
    y = torch.zeros(3, 3, dtype=torch.float16, device=dev)
    calls = {
        "rms_norm": [(lambda a: rms_norm(a, w), x), (lambda a: rms_norm(x, a), w),
                     (lambda a: rms_norm(x, w, residual=a), x)],
        "rms_norm_quantize": [(lambda a: rms_norm_quantize(a, w), x),
                              (lambda a: rms_norm_quantize(x, w, residual=a), x)],
        "dequantize_tokens": [(lambda a: dequantize_tokens(codes, a), w[:3]),
                              (lambda a: dequantize_tokens(codes, w[:3], a), w[:3])],
        "rotary": [(lambda a: rotary(a, x[:, None], p), x[:, None]),
                   (lambda a: rotary(x[:, None], a, p), x[:, None]),
                   (lambda a: rotary(a, None, p), x[:, None])],
        "adapters": [(lambda a: set_(a, index), half), (lambda a: set_(half, index, base=a), y),
                     (lambda a: set_.add_(y.clone(), a, index), half)]}[what]
    for call, t in calls:
        with forward_ad.dual_level():
            call(t)
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="tangent|forward-mode"):
                call(dual)
            call(forward_ad.unpack_dual(dual).primal)
