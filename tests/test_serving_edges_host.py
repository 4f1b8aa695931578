"""CPU: what a user's program can do around the operators of a quantized layer without
a launch: casts of a model, replaced buffers, exports that are not 8-bit codes."""
import ast
import glob
import os

import pytest
import torch

import g2ptq_amd
from g2ptq_amd import Int8Linear, PagedKVCache, _lib
from oracle import pack


def on_cpu(rows=5, columns=20, asym=True, bias=True):
    """An Int8Linear whose buffers are on the CPU (where it cannot be made or called)."""
    lin = Int8Linear.__new__(Int8Linear)
    torch.nn.Module.__init__(lin)
    lin.out_features, lin.in_features, lin._shape = rows, columns, (rows, 256)
    lin.sym = not asym
    g = torch.Generator().manual_seed(1)
    lin.register_buffer("weight", torch.randint(-128, 128, (rows, 256), generator=g,
                                                dtype=torch.int8))
    lin.register_buffer("weight_scale", torch.rand(rows, generator=g))
    lin.register_buffer("weight_sum", lin.weight.sum(1, dtype=torch.int32) if asym else None)
    lin.register_buffer("bias", torch.randn(rows, generator=g) if bias else None)
    return lin


CASTS = [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
         lambda m: m.type(torch.float16), lambda m: m.half().float()]


@pytest.mark.parametrize("cast", CASTS)
@pytest.mark.parametrize("asym,bias", [(True, True), (False, False)])
def test_a_cast_of_the_model_leaves_the_operands_as_they_are(cast, asym, bias):
    lin = on_cpu(asym=asym, bias=bias)
    before = {n: None if b is None else b.clone() for n, b in lin._buffers.items()}
    model = cast(torch.nn.Sequential(torch.nn.Linear(20, 20), lin))
    assert model[1] is lin
    for name, was in before.items():
        now = lin._buffers[name]
        assert (now is None) == (was is None), name
        if was is not None:
            assert now.dtype is was.dtype and torch.equal(now, was), name
    lin._operands()


def test_moves_still_follow_the_model():
    lin = on_cpu()
    assert all(b.device.type == "meta" for b in lin.to("meta", torch.float16)._buffers.values())
    assert lin.weight_scale.dtype is torch.float32


@pytest.mark.parametrize("name,make", [
    ("weight", lambda t: t.half()), ("weight", lambda t: t[:, :128].contiguous()),
    ("weight", lambda t: t.reshape(-1, 128)), ("weight", lambda t: t.t().contiguous().t()),
    ("weight", lambda t: t[:-1]), ("weight_scale", lambda t: t.bfloat16()),
    ("weight_scale", lambda t: t[:-1]), ("weight_scale", lambda t: t[:1].expand(5)),
    ("bias", lambda t: t.half()),
    ("bias", lambda t: torch.stack([t, t], 1)[:, 0]), ("weight_sum", lambda t: t.long())])
def test_replaced_buffers_are_refused_before_a_launch(name, make):
    lin = on_cpu()
    setattr(lin, name, make(getattr(lin, name)))
    with pytest.raises(ValueError, match=name + " is"):
        lin._operands()


def test_a_checkpoint_of_another_type():
    lin = on_cpu()
    state = {k: v.half() if v.is_floating_point() else v for k, v in lin.state_dict().items()}
    other = on_cpu()
    other.load_state_dict(state)  # copied into the fp32 buffers
    other._operands()
    other.load_state_dict(state, assign=True)
    with pytest.raises(ValueError, match="weight_scale is torch.float16"):
        other._operands()


def test_memory_that_kernels_read_has_its_type_from_the_code():
    """The kernels read and write fp32 by address: under torch.set_default_dtype with a
    16-bit type, memory without a type of its own would be half as large as they take it for."""
    allocators = ("empty", "zeros", "ones", "full", "rand", "randn")
    for path in sorted(glob.glob(os.path.join(os.path.dirname(g2ptq_amd.__file__), "*.py"))):
        with open(path) as f:
            tree = ast.parse(f.read())
        for call in ast.walk(tree):
            if (isinstance(call, ast.Call) and isinstance(call.func, ast.Attribute)
                    and isinstance(call.func.value, ast.Name) and call.func.value.id == "torch"
                    and call.func.attr in allocators):
                given = {k.arg for k in call.keywords}
                assert "device" not in given or "dtype" in given, (path, call.lineno)


def exported(bits, columns, rows=6):
    g = torch.Generator().manual_seed(bits)
    codes = torch.randint(-2 ** (bits - 1), 2 ** (bits - 1), (rows, columns), generator=g).float()
    return pack.compress((rows, columns), torch.float32, torch.full((rows, columns), 0.01), codes,
                         bits, columns)


@pytest.mark.parametrize("bits,columns", [(7, 64), (7, 130), (7, 4), (6, 4), (5, 3), (4, 2), (7, 1)])
def test_exports_of_fewer_bits_with_as_many_words_are_refused(bits, columns):
    wide, narrow = exported(8, columns), exported(bits, columns)
    assert narrow["weight_packed"].shape == wide["weight_packed"].shape
    with pytest.raises(ValueError, match="8-bit codes"):
        Int8Linear.from_export(narrow)
    with pytest.raises(ValueError, match="no 8-bit codes"):
        Int8Linear.from_export(wide, bits=bits)
    for kw in ({}, {"bits": 8}):  # past the checks of the codes
        with pytest.raises(RuntimeError, match="GPU"):
            Int8Linear.from_export(wide, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        Int8Linear.from_export(narrow, bits=8)


def test_a_layer_knows_what_was_exported_from_it():
    for grid, match in (((7, True), "codes of 7 bits"), ((8, False), "zero points")):
        layer = torch.nn.Linear(64, 6)
        layer._export_qparams, layer._export_grid = exported(8, 64), grid
        with pytest.raises(ValueError, match=match):
            Int8Linear.from_export(layer)


def test_products_that_no_launch_can_hold_are_refused():
    """More than 2^32 threads: the runtime would run what is left modulo 2^32."""
    lib, fake = _lib.load(), 4096
    for T, N in ((1, 1 << 28), (20, 1 << 29), (1 << 20, 1 << 20), ((1 << 22) - 1, 1 << 18)):
        assert lib.g2ptq_int8_linear(None, fake, 0, T, 64, 64, 1, fake, 256, fake, None, None, N,
                                     fake, N, None, 0) == -1
        assert b"too many" in lib.g2ptq_last_error()
        assert lib.g2ptq_int8_gemm(None, fake, 64, fake, None, fake, 256, fake, None, None, T, N,
                                   64, fake, 0, N, None, 0) == -1
        assert b"too many" in lib.g2ptq_last_error()


def test_a_cache_that_no_call_takes_is_not_made():
    for pages, page, heads in ((1 << 20, 64, 32), (1 << 31, 1, 1), (1 << 12, 4096, 128)):
        with pytest.raises(ValueError, match="2\\^31"):
            PagedKVCache(pages, page, heads, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCache((1 << 19) - 1, 64, 64, 64, device="cpu")


def test_sizes_stated_too_small_do_not_ask_for_all_memory():
    """A million tokens where max_q says eight: partial results of every share of every token
    would be half a TiB.  Sizes stated right are as before."""
    def size(*a):
        return _lib.query_size("g2ptq_paged_attention_workspace", *a)
    assert size(1 << 20, 32, 8, 128, 1, 8, 131072) <= 1 << 30
    assert size(8192, 32, 8, 128, 1, 5, 131072) <= 1 << 30
    assert size(512, 32, 8, 128, 1, 512, 2048) == 512 * 32 * 4 * 132 * 4
    assert size(1, 32, 8, 128, 1, 1, 4096) == 8 * 16 * 16 * 132 * 4
