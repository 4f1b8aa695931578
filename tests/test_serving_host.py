"""CPU: the host side of running a quantized layer: argument errors of the C entry
points (each returns before it touches a device), size queries, refusals of the Python
layer, and the oracle's grid against the weight quantizer's oracle."""
import ctypes

import pytest
import torch

from g2ptq_amd import Int8Linear, PagedKVCache, _lib, int8_matmul, quantize_tokens
from oracle import quant, serving

FAKE = 4096  # a 16-byte aligned address that no call here may follow


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cache(**kw):
    fields = dict(k_codes=FAKE, v_codes=FAKE, k_scale=FAKE, v_scale=FAKE, k_zero=None, v_zero=None,
                  flags=FAKE, pages=4, heads=2, page=16, dim=64, bits=8, sym=1)
    fields.update(kw)
    return _lib.KvCacheStruct(*(fields[n] for n, _ in _lib.KvCacheStruct._fields_))


@pytest.mark.parametrize("bad", [
    {"bits": 3}, {"bits": 16}, {"dim": 8}, {"dim": 72}, {"dim": 272}, {"page": 0}, {"page": 24},
    {"page": 8192}, {"heads": 0}, {"pages": -1}, {"flags": None}, {"k_codes": None},
    {"v_scale": None}, {"k_codes": FAKE + 8}, {"sym": 0}, {"pages": 1 << 30}], ids=str)
def test_cache_descriptions_are_checked(lib, bad):
    c = cache(**bad)
    assert lib.g2ptq_kv_write(None, ctypes.byref(c), FAKE, 1, 1, FAKE, 1, 1, 0, 3, FAKE) == -1
    assert b"kv_write" in lib.g2ptq_last_error()
    assert lib.g2ptq_kv_read(None, ctypes.byref(c), FAKE, 1, 1, 1, FAKE, 3, FAKE, FAKE, 0) == -1
    assert lib.g2ptq_paged_attention(None, ctypes.byref(c), FAKE, 128, 64, 0, 1, 2, FAKE, 1, 1, 1,
                                     FAKE, FAKE, 1, 16, 1.0, FAKE, None, 0) == -1
    assert b"paged_attention" in lib.g2ptq_last_error()


def test_cache_calls_check_their_arguments(lib):
    c = ctypes.byref(cache())
    for args in ((None, c, FAKE, 1, 1, FAKE, 1, 1, 3, 3, FAKE),      # dtype
                 (None, c, None, 1, 1, FAKE, 1, 1, 0, 3, FAKE),      # no keys
                 (None, c, FAKE, 1, 1, FAKE, 1, 1, 0, 3, None),      # no slots
                 (None, c, FAKE, 1, 1, FAKE, 1, 1, 0, 1 << 31, FAKE),
                 (None, None, FAKE, 1, 1, FAKE, 1, 1, 0, 3, FAKE)):
        assert lib.g2ptq_kv_write(*args) == -1
    for args in ((None, c, FAKE, 1, 1, 2, FAKE, 3, FAKE, FAKE, 0),   # row stride below width
                 (None, c, FAKE, 1, 1, 1, FAKE, 3, FAKE + 4, FAKE, 0),
                 (None, c, FAKE, 1, 1, 1, None, 3, FAKE, FAKE, 0),
                 (None, c, FAKE, 1, 1, 1, FAKE, -1, FAKE, FAKE, 0)):
        assert lib.g2ptq_kv_read(*args) == -1
    ok = [None, c, FAKE, 128, 64, 0, 1, 2, FAKE, 1, 1, 1, FAKE, FAKE, 1, 16, 1.0, FAKE, None, 0]
    for at, value in ((5, 2), (7, 3), (7, 0), (2, None), (8, None), (12, None), (13, None),
                      (17, None), (17, FAKE + 8), (9, 0), (14, 2), (15, -1), (10, 65535),
                      (11, 1 << 31)):
        args = list(ok)
        args[at] = value
        assert lib.g2ptq_paged_attention(*args) == -1, (at, value)
    # nothing to do: no device is touched
    assert lib.g2ptq_kv_write(None, c, None, 1, 1, None, 1, 1, 0, 0, None) == 0
    assert lib.g2ptq_kv_read(None, c, FAKE, 1, 1, 1, FAKE, 0, None, None, 0) == 0
    # shares of a long context need a workspace
    long = list(ok)
    long[9] = long[11] = 1024
    long[15] = 16384
    assert lib.g2ptq_paged_attention(*long) == -3


def test_linear_calls_check_their_arguments(lib):
    q = [None, FAKE, 0, 2, 64, 64, 1, FAKE, 64, FAKE, None]
    for at, value in ((2, 3), (4, 0), (4, 65537), (5, 63), (1, None), (7, None), (8, 72), (8, 48),
                      (7, FAKE + 8), (9, None), (6, 0), (3, -1), (3, 1 << 22)):
        args = list(q)
        args[at] = value
        assert lib.g2ptq_quantize_tokens(*args) == -1, (at, value)
    g = [None, FAKE, 64, FAKE, None, FAKE, 256, FAKE, None, None, 2, 8, 64, FAKE, 0, 8, None, 0]
    for at, value in ((2, 48), (2, 72), (2, 1 << 20), (1, None), (3, None), (4, FAKE), (5, None),
                      (6, 64), (6, 264), (7, None), (12, 65537), (13, None), (14, 5), (15, 7)):
        args = list(g)
        args[at] = value
        assert lib.g2ptq_int8_gemm(*args) == -1, (at, value)
    x = [None, FAKE, 0, 6, 64, 64, 1, FAKE, 256, FAKE, None, None, 8, FAKE, 8, None, 0]
    for at, value in ((1, None), (2, 4), (4, 0), (5, 10), (6, 0), (7, FAKE + 4), (9, None),
                      (13, None), (14, 4)):
        args = list(x)
        args[at] = value
        assert lib.g2ptq_int8_linear(*args) == -1, (at, value)
    assert lib.g2ptq_int8_linear(*x) == -3  # six tokens need a workspace
    x[3] = 0
    assert lib.g2ptq_int8_linear(*x) == 0


def test_workspace_sizes(lib):
    assert _lib.query_size("g2ptq_int8_linear_workspace", 1, 4096, 4096) == 0  # one launch
    big = _lib.query_size("g2ptq_int8_linear_workspace", 512, 4096, 4096)
    assert big >= 512 * (4096 + 8)
    assert _lib.query_size("g2ptq_int8_gemm_workspace", 512, 4096, 4096) == 0
    one = _lib.query_size("g2ptq_paged_attention_workspace", 1, 32, 8, 128, 1, 1, 4096)
    assert one >= 32 * 128 * 4 * 2
    assert _lib.query_size("g2ptq_paged_attention_workspace", 2048, 32, 8, 128, 1, 2048, 64) == 0
    fast = _lib.fastcall()
    assert fast.paged_attention_workspace(1, 32, 8, 128, 1, 1, 4096) == one
    assert fast.int8_linear_workspace(512, 4096, 4096) == big
    assert fast.int8_linear_workspace(512, 4096, 0) == -1
    with pytest.raises(ValueError, match="int8_linear_workspace"):
        _lib.workspace_fast("int8_linear_workspace", 512, 4096, 0)


def test_fast_calls_report_like_the_others(lib):
    c = cache(bits=3)
    fast = _lib.fastcall()
    with pytest.raises(TypeError, match="11 arguments"):
        fast.kv_write(0, 1)
    with pytest.raises(ValueError, match="kv_write"):
        _lib.call_fast("kv_write", 0, ctypes.addressof(c), FAKE, 1, 1, FAKE, 1, 1, 0, 3, FAKE)
    with pytest.raises(ValueError, match="int8_linear"):
        _lib.call_fast("int8_linear", 0, FAKE, 9, 6, 64, 64, 1, FAKE, 256, FAKE, None, None, 8, FAKE,
                       8, None, 0)


def test_without_the_fast_calls_the_same_entry_points_run(lib, monkeypatch):
    monkeypatch.setattr(_lib, "_FAST", False)
    c = cache(bits=3)
    with pytest.raises(ValueError, match="kv_read"):
        _lib.call_fast("kv_read", 0, ctypes.addressof(c), FAKE, 1, 1, 1, FAKE, 3, FAKE, FAKE, 0)
    with pytest.raises(ValueError, match="int8_linear"):
        _lib.call_fast("int8_linear", 0, FAKE, 9, 6, 64, 64, 1, FAKE, 256, FAKE, None, None, 8, FAKE,
                       8, None, 0)
    assert _lib.workspace_fast("int8_linear_workspace", 1, 4096, 4096) == 0


def test_the_python_layer_takes_gpu_tensors_only():
    codes = torch.zeros(4, 8, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="GPU"):
        Int8Linear(codes, torch.ones(4))
    with pytest.raises(ValueError, match="int8 codes"):
        Int8Linear(codes.float(), torch.ones(4))
    with pytest.raises(ValueError, match="one scale"):
        Int8Linear(codes, torch.ones(3))
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_tokens(torch.zeros(2, 8))
    with pytest.raises(NotImplementedError):
        quantize_tokens(torch.zeros(2, 8, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCache(4, 16, 2, 64, device="cpu")
    for args in ((4, 24, 2, 64), (4, 16, 2, 40), (4, 16, 0, 64), (-1, 16, 2, 64)):
        with pytest.raises(ValueError):
            PagedKVCache(*args, device="cpu")
    with pytest.raises(ValueError, match="4 or 8 bits"):
        PagedKVCache(4, 16, 2, 64, bits=5, device="cpu")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("sym", [True, False])
def test_the_oracles_grid_is_the_weight_quantizers(bits, sym):
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(50, 96, generator=g) * torch.exp(torch.randn(50, 1, generator=g))
    x[3] = x[3].abs()
    x[4] = -x[4].abs()
    codes, scale, zero = serving.quantize(x, bits, sym)
    s, z = quant.find_params(x, bits, sym)[:2]
    assert torch.equal(scale, s.reshape(-1)) and torch.equal(zero, z.reshape(-1))
    assert bool((codes >= -2 ** (bits - 1)).all()) and bool((codes < 2 ** (bits - 1)).all())
    err = (serving.dequantize(codes, scale, zero) - x.double()).abs()
    # half a step; the zero point's own rounding can cost the ends of the range another
    assert bool((err <= (0.501 if sym else 1.001) * scale.double()[:, None]).all())
