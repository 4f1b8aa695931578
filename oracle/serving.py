"""Oracle: running a quantized layer (test infrastructure only).

The token / cache grid restated in torch-CPU fp32, in the order of operations
that defines its codes, and the products and the attention in fp64.
"""
import math

import torch


def quantize(x, bits, sym):
    """(codes, scale, zero) of the groups along the last axis of ``x``: the weight
    quantizer's grid (utils/quant_utils.py:8-68) with one group per token.  A
    group of zeros has scale, codes and zero point 0; a non-finite scale goes
    with codes and zero point 0."""
    x = x.float()
    maxq = 2 ** (bits - 1) - 1
    minq = -(maxq + 1)
    if sym:
        scale = x.abs().amax(dim=-1) / torch.tensor((maxq - minq) / 2)
        zero = torch.zeros_like(scale)
    else:
        lo = torch.minimum(x.amin(dim=-1), torch.tensor(0.0))
        hi = torch.maximum(x.amax(dim=-1), torch.tensor(0.0))
        scale = (hi - lo) / torch.tensor(float(maxq - minq))
        zero = torch.clamp(torch.round(minq - lo / scale), minq, maxq)
    codes = torch.clamp(torch.round(x / scale[..., None]) + zero[..., None], minq, maxq)
    usable = torch.isfinite(scale) & (scale > 0)
    zero = torch.where(usable, zero, torch.zeros_like(zero))
    return torch.where(usable[..., None], codes, torch.zeros_like(codes)), scale, zero


def dequantize(codes, scale, zero):
    return scale[..., None].double() * (codes - zero[..., None]).double()


def linear(codes, scale, zero, weight, wscale, bias):
    """fp64 result and the magnitude of its terms before the last rounding."""
    acc = (codes - zero[..., None]).double() @ weight.double().T
    y = acc * scale.double()[..., None] * wscale.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def attention(q, k, v, cu_q, kv_lens, scale, v_span):
    """Causal attention in fp64.  ``k``, ``v``: per sequence (kv_len, heads, dim);
    ``v_span``: per sequence (kv_len, heads), the span of the values' grid
    (scale times its number of steps).

    Returns the output (zero outside the sequences and for queries without
    keys), Σ p·|v| per output element, per (query, head) the largest
    Σ|q·k|·scale over its keys and the largest span of their values, and per
    query its count of keys."""
    T, heads, dim = q.shape
    out = torch.zeros(T, heads, dim, dtype=torch.float64)
    size, logit = torch.zeros_like(out), torch.zeros(T, heads, dtype=torch.float64)
    count, span = torch.zeros(T, dtype=torch.int64), torch.zeros_like(logit)
    for b, n_kv in enumerate(kv_lens):
        q0, q1 = cu_q[b], cu_q[b + 1]
        for i in range(q0, q1):
            n = n_kv - (q1 - q0) + (i - q0) + 1
            if n <= 0:
                continue
            count[i] = n
            group = heads // k[b].shape[1]
            kk = k[b][:n].double().repeat_interleave(group, dim=1)
            vv = v[b][:n].double().repeat_interleave(group, dim=1)
            terms = q[i].double()[None] * kk
            p = torch.softmax(terms.sum(-1) * scale, dim=0)[..., None]
            out[i], size[i] = (p * vv).sum(0), (p * vv.abs()).sum(0)
            logit[i] = terms.abs().sum(-1).amax(0) * abs(scale)
            span[i] = v_span[b][:n].double().amax(0).repeat_interleave(group)
    return out, size, logit, span, count


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def linear_bound(dtype, y, size):
    """The integer sum is exact: its conversion, two products and a sum in fp32
    round once each (four units of 2^-24 of the terms), then the result rounds
    to ``dtype`` (its unit, or half a step of fp16's subnormals)."""
    inner = 4 * 2.0 ** -24 * size
    return inner + UNIT[dtype] * (y.abs() + inner) + TINY[dtype]


def attention_bound(dtype, out, size, logit, span, count, dim):
    """Error of an output element, to first order, each part of Σ p·|v| (size):

    - weights p·scale are rounded to 11 significant bits before the products
      with the values: 2^-11;
    - a logit's fp32 sum of dim products and its scaling: (dim + 4)·2^-24 of
      Σ|q·k|; the query's conversion to a scaled fp16 row is exact, but for elements
      below 2^-32 of the largest of a bf16 row, which move by at most 2^-40 of it:
      another 2^-24·dim of Σ|q·k| is there for them.  A logit's error changes p, and
      through the sum every other p: twice;
    - exp2, its argument's rounding (2^-24 of the logit, counted above) and the
      joining of partial results: 16 units of 2^-24;
    - fp32 sums over ``count`` keys, numerator and denominator: 2·count·2^-24;
    - weights p·scale below the normal range of fp16 lose their relative
      precision: they are held relative to a power of two above the largest scale
      and at most twice it, times 2^15, so they move by at most half of
      2^-24·2^-15 of twice the largest scale each, times the steps of the grid:
      count·2^-39·span (the sum that divides is at least 1);
    - then the rounding to ``dtype``.
    """
    part = (2.0 ** -11 + 16 * 2.0 ** -24 + 2 * count.double()[:, None] * 2.0 ** -24
            + 2 * (2 * dim + 4) * 2.0 ** -24 * logit)
    lost = count.double()[:, None] * 2.0 ** -39 * span
    inner = part[..., None] * size + lost[..., None]
    return inner + UNIT[dtype] * (out.abs() + inner) + TINY[dtype]


def slot_map(table, page, cu, kv_lens):
    """Slots of every sequence's last ``cu[b+1] − cu[b]`` tokens of ``kv_lens[b]``."""
    slots = []
    for b, n in enumerate(kv_lens):
        for p in range(n - (cu[b + 1] - cu[b]), n):
            slots.append(int(table[b][p // page]) * page + p % page)
    return torch.tensor(slots, dtype=torch.int64)


def default_scale(dim):
    return 1.0 / math.sqrt(dim)
