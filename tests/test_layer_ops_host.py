"""CPU: the host side of norms, rotary positions, page tables and low-rank adapters: argument
errors of the C entry points (each returns before it touches a device), size queries, the
fast-call bindings, refusals of the Python layer, frequencies, and the oracles."""
import ctypes
import math
import weakref

import pytest
import torch

from g2ptq_amd import (LowRankAdapters, PageTables, Rotary, _lib, dequantize_tokens, rms_norm,
                       rms_norm_quantize, rotary_frequencies)
from g2ptq_amd.norm_utils import _rows
from oracle import layer_ops

FAKE = 4096  # a 16-byte aligned address that no call here may follow


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def tables(**kw):
    fields = dict(table=FAKE, lengths=FAKE, free_pages=FAKE, free_count=FAKE, mark=FAKE, flags=FAKE,
                  seqs=4, width=8, pages=10, page=16)
    fields.update(kw)
    return _lib.PageTablesStruct(*(fields[n] for n, _ in _lib.PageTablesStruct._fields_))


def adapters(**kw):
    fields = dict(down=FAKE, up=FAKE, rank=FAKE, scale=FAKE, flags=FAKE, n=2, R=16, K=64, N=64,
                  dtype=0)
    fields.update(kw)
    return _lib.AdapterSetStruct(*(fields[n] for n, _ in _lib.AdapterSetStruct._fields_))


def test_norm_checks_its_arguments(lib):
    good = [None, FAKE, 64, 0, None, 0, 0, 0, FAKE, 0, 3, 1, 64, 1e-6, FAKE, None, 1, None, 0, None,
            None]
    for at, value in ((1, None), (7, 3), (7, -1), (8, None), (9, 3), (10, -1), (11, 0), (12, 0),
                      (12, 65537), (13, -1.0), (13, math.nan), (13, math.inf), (14, None)):
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_rms_norm(*bad) == -1, at
        assert b"rms_norm" in lib.g2ptq_last_error()
    good[17:] = [FAKE, 64, FAKE, FAKE]
    for at, value in ((17, FAKE + 8), (18, 63), (18, 48), (19, None)):
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_rms_norm(*bad) == -1, at
    bad = list(good)
    bad[16], bad[20] = 0, None  # zero points of the asymmetric grid
    assert lib.g2ptq_rms_norm(*bad) == -1
    good[10] = 0
    assert lib.g2ptq_rms_norm(*good) == 0  # no rows, no launch
    for args in ((None, FAKE, 64, FAKE, None, 3, 64, FAKE, 3), (None, None, 64, FAKE, None, 3, 64,
                 FAKE, 0), (None, FAKE, 64, None, None, 3, 64, FAKE, 0),
                 (None, FAKE, 64, FAKE, None, 3, 65537, FAKE, 0),
                 (None, FAKE, 64, FAKE, None, -1, 64, FAKE, 0),
                 (None, FAKE, 64, FAKE, None, 3, 64, None, 0)):
        assert lib.g2ptq_dequantize_tokens(*args) == -1
        assert b"dequantize_tokens" in lib.g2ptq_last_error()
    assert lib.g2ptq_dequantize_tokens(None, None, 0, None, None, 0, 64, None, 0) == 0


def test_rotary_checks_its_arguments(lib):
    good = [None, FAKE, 128, 64, 2, FAKE, 64, 64, 1, 0, 3, 64, 64, 0, FAKE, FAKE, 1.0, FAKE, FAKE]
    for at, value in ((1, None), (4, -1), (4, 65536), (5, None), (8, 65536), (9, 3), (10, -1),
                      (11, 62), (11, 1026), (12, 0), (12, 63), (12, 66), (14, None), (15, None),
                      (17, None), (18, None)):
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_rotary(*bad) == -1, at
        assert b"rotary" in lib.g2ptq_last_error()
    good[10] = 0
    assert lib.g2ptq_rotary(*good) == 0


@pytest.mark.parametrize("bad", [
    {"seqs": 0}, {"width": 0}, {"pages": -1}, {"pages": 1 << 31}, {"page": 0}, {"page": 24},
    {"page": 8192}, {"width": 1 << 28}, {"table": None}, {"lengths": None}, {"free_pages": None},
    {"free_count": None}, {"mark": None}, {"flags": None}], ids=str)
def test_page_tables_are_checked(lib, bad):
    t = ctypes.byref(tables(**bad))
    assert lib.g2ptq_pages_extend(None, t, FAKE, FAKE, 2, 3, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                  4096) == -1
    assert b"pages_extend" in lib.g2ptq_last_error()
    assert lib.g2ptq_pages_release(None, t, FAKE, None, 2, FAKE, 4096) == -1
    assert b"pages_release" in lib.g2ptq_last_error()


def test_page_calls_check_their_arguments(lib):
    t = ctypes.byref(tables())
    good = [None, t, FAKE, FAKE, 2, 3, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4096]
    for at, value in ((1, None), (2, None), (3, None), (4, -1), (4, (1 << 20) + 1), (5, -1),
                      (5, 1 << 31), (6, None), (7, None), (8, None), (9, None), (10, None),
                      (11, FAKE + 2)):
        bad = list(good)
        bad[at] = value
        if at == 4 and value > 0:
            bad[12] = 1 << 30
        assert lib.g2ptq_pages_extend(*bad) == -1, at
    for at, value in ((11, None), (12, 39)):  # two requests of 20 bytes each
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_pages_extend(*bad) == -3, at
    assert lib.g2ptq_pages_release(None, t, FAKE, None, 2, FAKE, 39) == -3
    assert lib.g2ptq_pages_release(None, t, None, None, 2, FAKE, 4096) == -1
    assert lib.g2ptq_pages_release(None, t, None, None, 0, None, 0) == 0
    assert _lib.query_size("g2ptq_pages_workspace", 2) == 40
    assert _lib.fastcall().pages_workspace(1000) == 20000
    for n in (-1, (1 << 20) + 1):
        with pytest.raises(ValueError, match="pages_workspace"):
            _lib.workspace_fast("pages_workspace", n)


@pytest.mark.parametrize("bad", [
    {"dtype": 2}, {"dtype": -1}, {"n": 0}, {"K": 0}, {"K": (1 << 20) + 1}, {"N": 0}, {"R": 8},
    {"R": 24}, {"R": 528}, {"down": None}, {"up": None}, {"rank": None}, {"scale": None},
    {"flags": None}, {"down": FAKE + 8}, {"up": FAKE + 2}], ids=str)
def test_adapter_sets_are_checked(lib, bad):
    a = ctypes.byref(adapters(**bad))
    assert lib.g2ptq_adapters(None, a, FAKE, 64, FAKE, 3, FAKE, 64, FAKE, 64, FAKE, 1 << 20) == -1
    assert b"adapters" in lib.g2ptq_last_error()


def test_adapter_calls_check_their_arguments(lib):
    a = ctypes.byref(adapters())
    good = [None, a, FAKE, 64, FAKE, 3, FAKE, 64, FAKE, 64, FAKE, 1 << 20]
    for at, value in ((1, None), (2, None), (4, None), (5, -1), (5, 1 << 31), (8, None),
                      (10, FAKE + 8)):
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_adapters(*bad) == -1, at
    need = _lib.query_size("g2ptq_adapters_workspace", 3, 64, 2, 16)
    assert need == 3 * 16 * 4 == _lib.fastcall().adapters_workspace(3, 64, 2, 16)
    for at, value in ((10, None), (11, need - 1)):
        bad = list(good)
        bad[at] = value
        assert lib.g2ptq_adapters(*bad) == -3, at
    good[5] = 0
    assert lib.g2ptq_adapters(*good) == 0
    # more shares of K where tokens are few and columns many, never more than eight
    sizes = [_lib.query_size("g2ptq_adapters_workspace", 1, K, 4, 16) // 64
             for K in (64, 1024, 4096, 1 << 20)]
    assert sizes == sorted(sizes) and sizes[0] == 1 and 1 < sizes[-1] <= 8


def test_fast_calls_and_their_fallback(lib, monkeypatch):
    fast = _lib.fastcall()
    for name, n in (("rms_norm", 21), ("dequantize_tokens", 9), ("rotary", 19),
                    ("pages_workspace", 1), ("pages_extend", 13), ("pages_release", 7),
                    ("adapters_workspace", 4), ("adapters", 12)):
        with pytest.raises(TypeError, match=f"{name} takes {n} arguments"):
            getattr(fast, name)()
    t, a = tables(page=3), adapters(R=8)
    for fallback in (False, True):
        if fallback:
            monkeypatch.setattr(_lib, "_FAST", False)
        with pytest.raises(ValueError, match="pages_release.*3 slots"):
            _lib.call_fast("pages_release", 0, ctypes.addressof(t), FAKE, None, 2, FAKE, 4096)
        with pytest.raises(ValueError, match="adapters of 8 ranks"):
            _lib.call_fast("adapters", 0, ctypes.addressof(a), FAKE, 64, FAKE, 3, FAKE, 64, FAKE, 64,
                           FAKE, 1 << 20)
        with pytest.raises(ValueError, match="63 of 64 channels"):
            _lib.call_fast("rotary", 0, FAKE, 1, 1, 1, None, 0, 0, 0, 0, 3, 64, 63, False, FAKE, FAKE,
                           1.0, FAKE, None)
        assert _lib.workspace_fast("pages_workspace", 3) == 60


def test_the_python_layer_takes_gpu_tensors_only():
    x, w = torch.ones(3, 8), torch.ones(8)
    codes = torch.ones(3, 8, dtype=torch.int8)
    for call in (lambda: rms_norm(x, w), lambda: rms_norm_quantize(x, w),
                 lambda: dequantize_tokens(codes, w[:3]), lambda: Rotary(64, device="cpu"),
                 lambda: PageTables(4, 16, 2, 3, device="cpu"),
                 lambda: LowRankAdapters([x.bfloat16()], [torch.ones(5, 3).bfloat16()])):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError):
        rms_norm(torch.ones(()), w)
    with pytest.raises(NotImplementedError):
        rms_norm(x.long(), w)
    with pytest.raises(ValueError, match="down and"):
        LowRankAdapters([], [])
    for args in ((4, 24, 2, 2), (4, 16, 0, 2), (-1, 16, 2, 2), (4, 4096, 2, 1 << 19)):
        with pytest.raises(ValueError):
            PageTables(*args, device="cpu")


def test_rows_are_told_by_two_strides_or_copied():
    x = torch.arange(2 * 3 * 4 * 10.0).view(2, 3, 4, 10)
    views = [x, x[:, :, 1:3], x[:, 1], x[..., 2:], x.transpose(0, 2), x[0, 0, 0], x[:1, :, 2:3],
             x[:, :, :1].expand(2, 3, 5, 10), x.permute(3, 0, 1, 2), x[:0], x[:, :, 0], x[::2, :, ::2],
             x[:, :1, ::3, :7]]
    for v in views:
        t, rows, inner, outer_stride, inner_stride = _rows(v, "rows")
        C = v.shape[-1]
        flat = v.reshape(-1, C)
        assert rows == len(flat) and (inner == 1 or rows % inner == 0)
        for i in range(rows):
            at = i // inner * outer_stride + i % inner * inner_stride
            assert torch.equal(torch.as_strided(t, (C,), (1,), t.storage_offset() + at), flat[i])


def test_frequencies():
    theta, m = rotary_frequencies(64)
    assert theta.dtype is torch.float64 and m == 1.0
    torch.testing.assert_close(theta, 10000.0 ** (-torch.arange(0, 64, 2).double() / 64))
    long = {"type": "yarn", "factor": 32.0, "original_positions": 4096}
    theta2, m = rotary_frequencies(64, 10000.0, long)
    # the fastest pairs stay, the slowest are interpolated whole, in between they fall
    ratio = theta2 / theta
    assert ratio[0] == 1 and abs(float(ratio[-1]) - 1 / 32) < 1e-12
    assert bool((ratio.diff() <= 0).all()) and abs(m - (1 + 0.1 * math.log(32))) < 1e-12
    bands = {"type": "bands", "factor": 4.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_positions": 8192}
    ratio = rotary_frequencies(128, 500000.0, bands)[0] / rotary_frequencies(128, 500000.0)[0]
    assert ratio[0] == 1 and abs(float(ratio[-1]) - 0.25) < 1e-12
    assert bool((ratio.diff() <= 1e-15).all())
    before = torch.get_default_dtype()
    try:  # numbers stay numbers of 64 bits under any default type
        torch.set_default_dtype(torch.float16)
        torch.testing.assert_close(rotary_frequencies(64)[0], theta, rtol=0, atol=0)
    finally:
        torch.set_default_dtype(before)
    for bad in ({"type": "linear"}, {"factor": 2.0}, {"type": "linear", "factor": -1.0},
                {"type": "ntk", "factor": math.inf}, {"type": "bands", "factor": 2.0},
                {"type": "yarn", "factor": 2.0, "original_positions": 10, "beta_fast": 1,
                 "beta_slow": 2}, {"type": "bands", "factor": 2.0, "low_freq_factor": 4.0,
                                   "high_freq_factor": 1.0, "original_positions": 10}):
        with pytest.raises(ValueError):
            rotary_frequencies(64, 10000.0, bad)


def test_the_oracle_of_pages_keeps_every_page_once():
    import random
    r = random.Random(5)
    p = layer_ops.Pages(30, 4, 8, 6)
    for _ in range(300):
        rows = r.sample(range(8), r.randint(1, 8))
        before = (list(p.free), [list(x) for x in p.rows], list(p.lengths))
        if r.random() < 0.6:
            p.extend(rows, [r.randint(0, 9) for _ in rows], 100)
            if r.random() < 0.5:  # a release of what a step took restores the stack
                p.release(rows, [before[2][x] for x in rows])
                assert (p.free, p.rows, p.lengths) == before
        else:
            p.release(rows, [r.randint(0, p.lengths[x]) for x in rows])
        held = [x for row in p.rows for x in row]
        assert sorted(held + p.free) == list(range(30))
        assert all(len(x) == -(-n // 4) for x, n in zip(p.rows, p.lengths))


def test_calls_hold_their_workspace_until_they_return(monkeypatch):
    """The buffer of a call on the current stream is in the caller's hand at its launch: another
    thread's call may replace the cached one by a larger, and what is freed becomes somebody's
    output.  The Python layer's paths, on host tensors with the launch taken out."""
    held, launched = [], []

    def scratch(nbytes, device):
        buf = torch.empty(nbytes + 16, dtype=torch.uint8)
        held[:] = [weakref.ref(buf), buf.data_ptr()]
        return buf

    def launch(name, *args):
        launched.append(name)
        assert held[0]() is not None, f"{name}: the workspace was dropped before the launch"
        assert held[1] in args

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)  # (host tensors' device)
    monkeypatch.setattr(_lib, "current_stream", lambda: 0)
    monkeypatch.setattr(_lib, "require_current", lambda t, what: None)
    monkeypatch.setattr(_lib, "scratch", scratch)
    monkeypatch.setattr(_lib, "call_fast", launch)
    a = LowRankAdapters.__new__(LowRankAdapters)
    a.in_features, a.out_features, a.dtype = 64, 32, torch.bfloat16
    a.device, a._device, a._n, a._rank, a._address = torch.device("cpu"), -1, 2, 16, FAKE
    x, y = torch.ones(3, 64).bfloat16(), torch.ones(3, 32).bfloat16()
    index = torch.zeros(3, dtype=torch.int32)
    a(x, index, base=y)
    a(x, index)
    a.add_(y, x, index)
    t = PageTables.__new__(PageTables)
    t.device, t._device, t._address = torch.device("cpu"), -1, FAKE
    t.release(index)
    assert launched == ["adapters"] * 3 + ["pages_release"]


def test_a_check_of_page_tables_names_all_that_was_met():
    """Both kinds of flags at once: the error names both, since it clears both."""
    t = PageTables.__new__(PageTables)
    t._held = (None,) * 5 + (torch.zeros(1, dtype=torch.int32),)
    t.check()
    for flags, error, kinds in (
            (_lib.FLAG_BAD_INDEX, IndexError, ("a row outside",)),
            (_lib.FLAG_NO_ROOM, RuntimeError, ("no free page",)),
            (_lib.FLAG_BAD_INDEX | _lib.FLAG_NO_ROOM, IndexError, ("a row outside", "no free page"))):
        t.flags.fill_(flags)
        with pytest.raises(error) as raised:
            t.check()
        said = str(raised.value)
        for kind in ("a row outside", "no free page"):
            assert (kind in said) == (kind in kinds), said
        t.check()


def test_adapter_sets_say_whether_a_weight_is_infinite(lib):
    """The dtype's bit of its own passes the checks beside both types, and nothing else does."""
    for dtype, bad in ((4, False), (5, False), (6, True), (8, True), (12, True)):
        a = ctypes.byref(adapters(dtype=dtype))
        # (no tokens: no launch)
        status = lib.g2ptq_adapters(None, a, FAKE, 64, FAKE, 0, FAKE, 64, FAKE, 64, FAKE, 1 << 20)
        assert status == (-1 if bad else 0), dtype
