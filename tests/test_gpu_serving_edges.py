"""GPU: the operators of a quantized layer at the edges that a user's program reaches."""
import pytest
import torch

from oracle import serving
from tests._util import assert_bitexact, gen
from tests.test_gpu_int8_linear import _check, _tokens, _weights
from tests.test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sym", [True, False])
def test_casts_of_a_model_leave_its_int8_linears_right(dev, sym):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    w, wscale, bias = _weights(70, 130, 3)
    for T in (1, 40):
        x = _tokens(T, 130, torch.float16, T)
        rc, rs, rz = serving.quantize(x, 8, sym)
        for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                     lambda m: m.cpu().half().to(dev)):
            lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=sym)
            cast(torch.nn.Sequential(torch.nn.Linear(8, 8, device=dev), lin))
            y = lin(x.to(dev))
            _check(y, rc, rs, rz, w, wscale, bias, torch.float16)
            c, s, z = quantize_tokens(x.to(dev), sym=sym)
            assert_bitexact(int8_matmul(c, s, lin, zero=z, dtype=torch.float16), y, "apart")
    lin.load_state_dict({k: v.half() if v.is_floating_point() else v
                         for k, v in lin.state_dict().items()}, assign=True)
    for call in (lambda: lin(x.to(dev)), lambda: int8_matmul(c, s, lin, zero=z)):
        with pytest.raises(ValueError, match="weight_scale is torch.float16"):
            call()
    lin.load_state_dict(Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev),
                                   sym=sym).state_dict(), assign=True)
    lin.weight_scale = lin.weight_scale.cpu()
    with pytest.raises(ValueError, match="weight_scale is .* on cpu"):
        lin(x.to(dev))


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64], ids=str)
def test_torchs_default_type_changes_nothing(dev, default):
    from g2ptq_amd import GPTQGuided, G2PTQ, Int8Linear, PagedKVCache, int8_matmul, quantize_tokens
    from g2ptq_amd import paged_attention
    T, K, H, D, page = 40, 130, 2, 64, 16
    w, wscale, bias = _weights(70, K, 4)
    x = _tokens(T, K, torch.bfloat16, 5)
    k = _tokens(T, H * D, torch.float16, 6).view(T, H, D).to(dev)
    q = _tokens(T, 4 * D, torch.float16, 7).view(T, 4, D).to(dev)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    cu, lens = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([0, T], [T]))
    slots = serving.slot_map(table.cpu(), page, [0, T], [T]).to(dev)

    def serve():
        lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=False)
        c, s, z = quantize_tokens(x.to(dev), sym=False)
        cache = PagedKVCache(3, page, H, D, bits=4, sym=False, device=dev)
        cache.write(k, k, slots)
        return [c, s, z, lin(x.to(dev)), int8_matmul(c, s, lin, zero=z),
                *cache.read(table, cu, T), paged_attention(q, cache, table, cu, lens),
                cache.k_scale, cache.v_scale]

    ref = serve()
    layers = [torch.nn.Linear(64, 32, bias=False, device=dev)]
    sal = [torch.ones(1, 4, 1, device=dev)]
    was = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = serve()
        acts = (GPTQGuided(layers, sal, 1).act_square, G2PTQ(layers, [sal], [None], 1).act_square)
    finally:
        torch.set_default_dtype(was)
    for i, (a, b) in enumerate(zip(got, ref)):
        assert a.dtype is b.dtype
        assert_bitexact(a, b, f"output {i}")
    assert all(a.dtype is torch.float32 for a in acts)


@pytest.mark.parametrize("bits,sym,match", [(7, True, "codes of 7 bits"), (8, False, "zero points"),
                                            (8, True, None)])
def test_a_layer_knows_what_was_exported_from_it(dev, bits, sym, match):
    from g2ptq_amd import GPTQ, Int8Linear, WeightQuantizer, make_group_quantizers
    from g2ptq_amd.compressed_tensors_utils import register_qparam_buffers
    lin = torch.nn.Linear(64, 48, device=dev)
    gq = GPTQ([lin])
    q = WeightQuantizer()
    q.configure(bits, perchannel=True, sym=sym)
    gq.quantizer = make_group_quantizers(q, 64, -1)
    gq.add_batch(0, _tokens(256, 64, torch.float32, 1).to(dev).unsqueeze(0), None)
    gq.fasterquant(blocksize=32, percdamp=0.01, groupsize=-1, backend="hip",
                   export_compressed_tensors=True)
    for _ in range(2):
        if match:
            with pytest.raises(ValueError, match=match):
                Int8Linear.from_export(lin)
        else:
            run = Int8Linear.from_export(lin)
            assert_bitexact(run.weight[:, :64].float() * run.weight_scale[:, None], lin.weight,
                            "export")
        register_qparam_buffers([lin])


@pytest.mark.parametrize("sym", [True, False])
@pytest.mark.parametrize("shape", [(37,), (1, 37), (2, 3, 37), (0, 37), (0, 4, 37), (4, 0, 37)])
def test_tokens_of_any_shape(dev, shape, sym):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    x = _tokens(max(1, int(torch.tensor(shape[:-1]).prod())), 37, torch.float16, 8)
    x = x[:0].reshape(shape) if 0 in shape else x.reshape(shape)
    c, s, z = quantize_tokens(x.to(dev), sym=sym)
    assert c.shape == shape and s.shape == shape[:-1] and (z is None) == sym
    if x.numel():
        rc, rs, rz = serving.quantize(x, 8, sym)
        assert_bitexact(c.float(), rc, "codes")
        assert_bitexact(s, rs, "scale")
        assert sym or torch.equal(z.cpu(), rz)
    w, wscale, bias = _weights(20, 37, 9)
    lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=sym)
    y = int8_matmul(c, s, lin, zero=z, dtype=torch.float16)
    assert y.shape == shape[:-1] + (20,)
    assert_bitexact(y, lin(x.to(dev)), "linear")


def test_the_product_takes_tensors_of_one_device(dev):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    w, wscale, bias = _weights(20, 37, 9)
    lin = Int8Linear(w.to(dev), wscale.to(dev), bias=bias.to(dev), sym=False)
    c, s, z = quantize_tokens(_tokens(3, 37, torch.float16, 8).to(dev), sym=False)
    for scale, zero, name in ((s.cpu(), z, "scale"), (s, z.cpu(), "zero")):
        with pytest.raises(ValueError, match=f"{name} on cpu, codes on cuda"):
            int8_matmul(c, scale, lin, zero=zero)
    with pytest.raises(ValueError, match="weights on cpu"):
        int8_matmul(c, s, lin.cpu(), zero=z)
    with pytest.raises(ValueError, match="weights on cpu"):
        int8_matmul(c[:0], s[:0], lin, zero=z[:0])


@pytest.mark.parametrize("T", [3, 40])
def test_codes_with_rows_far_apart(dev, T):
    from g2ptq_amd import Int8Linear, int8_matmul, quantize_tokens
    w, wscale, _ = _weights(20, 4096, 9)
    lin = Int8Linear(w.to(dev), wscale.to(dev))
    c, s, _ = quantize_tokens(_tokens(T, 4096, torch.float16, 8).to(dev))
    ref = int8_matmul(c, s, lin)
    for pitch in ((1 << 20) - 16, 1 << 20, (1 << 20) + 4096):
        wide = torch.zeros(T, pitch, dtype=torch.int8, device=dev)
        wide[:, :4096] = c
        assert_bitexact(int8_matmul(wide[:, :4096], s, lin), ref, f"{pitch}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits,sym", [(8, True), (4, False)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [60]), ([3, 1], [90, 300]), ([70], [100])], ids=str)
def test_small_queries_beside_a_large_one(dev, q_lens, kv_lens, bits, sym, dtype):
    """One channel of the queries 2^24 above the others, where the keys are zero: the others
    alone make the logits, and the bound has the sum of |q k|, which has no part of it."""
    def edit(q, k, v, cu):
        q *= 2.0 ** -9
        q[:, :, 5] = 3e4
        k *= 30
        k[:, :, 5] = 0
    b = Batch(dev, q_lens, kv_lens, 4, 2, 64, 16, bits, sym, dtype, edit=edit)
    b.check(b.run())


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [1]), ([1], [700]), ([5, 2], [3, 400]),
                                            ([70], [70]), ([30, 200], [20, 900])], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_queries_without_a_finite_logit_are_nan(dev, bad, q_lens, kv_lens):
    """An infinite element makes every logit of its row infinite or NaN, and a softmax of
    those is NaN, also where all are -inf; rows without keys are zero all the same."""
    def edit(q, k, v, cu):
        q[::2, 1, 7] = bad
        k[:, :, 7] = k[:, :, 7].abs() + 0.5
        if bad < 0:
            q[::2, 1, 8], k[:, :, 8] = -bad, -k[:, :, 8].abs() - 0.5
    for kw in ({}, {"max_q": max(q_lens), "max_kv": max(kv_lens)}):
        b = Batch(dev, q_lens, kv_lens, 4, 2, 64, 16, 8, True, torch.bfloat16, edit=edit)
        got = b.run(**kw)
        rows = torch.zeros(got.shape[:2], dtype=torch.bool)
        rows[::2, 1] = True
        count = torch.cat([torch.arange(n - m + 1, n + 1) for m, n in zip(q_lens, kv_lens)])
        assert bool(got.cpu()[rows & (count > 0)[:, None]].isnan().all())
        assert bool((got.cpu()[count <= 0] == 0).all())
        good = Batch(dev, q_lens, kv_lens, 4, 2, 64, 16, 8, True, torch.bfloat16,
                     edit=lambda q, k, v, cu: (edit(q, k, v, cu), q.nan_to_num_(0, 0, 0)))
        keep = ~rows & (count > 0)[:, None]
        assert_bitexact(got.cpu()[keep], good.run(**kw).cpu()[keep], "other rows")


def test_tangents_are_refused_like_gradients(dev):
    from torch.autograd import forward_ad
    from g2ptq_amd import Int8Linear, PagedKVCache, paged_attention, quantize_tokens
    w, wscale, _ = _weights(20, 64, 9)
    lin = Int8Linear(w.to(dev), wscale.to(dev))
    cache = PagedKVCache(2, 16, 1, 64, device=dev)
    x = _tokens(3, 64, torch.float16, 8).to(dev)
    slots = torch.arange(3, device=dev)
    table, cu, lens = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([[0]], [0, 3], [3]))

    def calls(t):
        k = t.view(3, 1, 64)
        plain = x.view(3, 1, 64)
        return (lambda: lin(t), lambda: quantize_tokens(t), lambda: cache.write(k, plain, slots),
                lambda: cache.write(plain, k, slots),
                lambda: paged_attention(k, cache, table, cu, lens))

    for call in calls(x):
        call()
    ref = lin(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls(dual):
            with pytest.raises(RuntimeError, match="inference only"):
                call()
        assert_bitexact(lin(x), ref, "a tensor without a tangent")
        assert_bitexact(lin(forward_ad.unpack_dual(dual).primal), ref, "primal")


def test_many_sequences_without_stated_sizes(dev):
    """Without max_q every sequence is taken to have all tokens: 2^24 row tiles here, more
    threads than a launch can have."""
    from g2ptq_amd import PagedKVCache, paged_attention
    B, n, T = 8192, 32, 1 << 18
    k = _tokens(2 * n, 16, torch.float16, 1).view(2 * n, 1, 16).to(dev)
    cache = PagedKVCache(4, 16, 1, 16, device=dev)
    cache.write(k, k, torch.arange(2 * n, device=dev))
    q = _tokens(T, 16, torch.float16, 2).view(T, 1, 16).to(dev)
    # the sequences' keys: two texts, shared by all
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev).repeat(B // 2, 1)
    cu = torch.arange(0, T + 1, n, dtype=torch.int32, device=dev)
    lens = torch.full((B,), n, dtype=torch.int32, device=dev)
    out = paged_attention(q, cache, table, cu, lens)
    ref = paged_attention(q, cache, table, cu, lens, max_q=n, max_kv=n)
    assert_bitexact(out, ref, "stated sizes")
    cache.check()
    for b in (0, 1, B - 1):
        one = paged_attention(q[b * n:(b + 1) * n], cache, table[b:b + 1], cu[:2], lens[:1])
        assert_bitexact(out[b * n:(b + 1) * n], one, f"sequence {b}")


@pytest.mark.parametrize("bits,heads,kv_heads,dim", [(8, 4, 2, 64), (4, 3, 1, 128), (8, 2, 1, 256)])
def test_more_row_tiles_than_stated(dev, bits, heads, kv_heads, dim):
    """Workgroups take further tiles of rows in turn."""
    b = Batch(dev, [300, 40, 700], [500, 900, 700], heads, kv_heads, dim, 16, bits, False,
              torch.bfloat16)
    b.check(b.run(max_q=20), "one tile for six")
    b.check(b.run(max_q=260, max_kv=300), "some")


def test_joining_very_many_rows(dev):
    """Two sequences, the second's few rows in shares whose joined rows lie past 2^28."""
    from g2ptq_amd import PagedKVCache, paged_attention
    T, n, D = (1 << 28) + 4, 3000, 16
    k = _tokens(n, D, torch.float16, 1).view(n, 1, D).to(dev)
    cache = PagedKVCache(188, 16, 1, D, device=dev)
    cache.write(k, k, torch.arange(n, device=dev))
    q = _tokens(1, D, torch.float16, 2).view(1, 1, D).to(dev)
    table = torch.arange(188, dtype=torch.int32, device=dev).repeat(2, 1)
    i32 = dict(dtype=torch.int32, device=dev)
    out = paged_attention(q.expand(T, 1, D), cache, table, torch.tensor([0, T - 4, T], **i32),
                          torch.tensor([0, n], **i32))
    one = paged_attention(q.expand(4, 1, D), cache, table[:1], torch.tensor([0, 4], **i32),
                          torch.tensor([n], **i32))
    assert float(one.abs().min()) > 0
    torch.testing.assert_close(out[-4:], one, rtol=2 ** -9, atol=2 ** -9)
    assert float(out[:1 << 20].abs().max()) == 0 and float(out[-(1 << 20):-4].abs().max()) == 0


def test_writing_very_many_tokens(dev):
    """2^30 heads of tokens, four lanes each: more threads than a launch can have.  The last
    token is written like the first."""
    from g2ptq_amd import PagedKVCache
    H, D, T = 65535, 64, (1 << 30) // 65535 + 2
    cache = PagedKVCache(2, 1, H, D, device=dev)
    x = torch.linspace(-3, 5, D, device=dev)
    slots = torch.full((T,), -1, dtype=torch.int64, device=dev)
    slots[0], slots[-1] = 0, 1
    cache.write(x.expand(T, H, D), (x * 2).expand(T, H, D), slots)
    rc, rs, _ = serving.quantize(x.cpu(), 8, True)
    for codes, scale, f in ((cache.k_codes, cache.k_scale, 1), (cache.v_codes, cache.v_scale, 2)):
        assert bool((scale == float(rs) * f).all())
        assert bool((codes.float() - 128 == rc.to(dev)).all())


def test_reading_very_many_tokens(dev):
    """2^30 tokens and some, 64 to a workgroup: the last sequence lies past the first launch."""
    from g2ptq_amd import PagedKVCache
    T = (1 << 30) + 40
    cache = PagedKVCache(2, 64, 1, 16, bits=4, device=dev)
    x = _tokens(64, 16, torch.float16, 3).view(64, 1, 16).to(dev)
    cache.write(x, x, torch.arange(64, device=dev))
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 50], dtype=torch.int32, device=dev)
    first = cache.read(table, cu, 50, dtype=torch.float16)
    for b in range(2):  # the first rows, then the last
        cu = torch.tensor([0, 50] if b == 0 else [T - 50, T], dtype=torch.int32, device=dev)
        k, v = cache.read(table, cu, T, dtype=torch.float16)
        for got, ref in zip((k, v), first):
            assert_bitexact(got[:50] if b == 0 else got[-50:], ref, "rows")
            rest = got[50:] if b == 0 else got[:-50]
            assert all(not bool(rest[i:i + (1 << 24)].any())
                       for i in range(0, len(rest), 1 << 27)) and not bool(rest[-1000:].any())
        del k, v, got, rest
    torch.cuda.empty_cache()
