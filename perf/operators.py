"""Performance cases of the operators that run a quantized layer.

``op`` of a case:

- ``linear``     a linear with 8-bit weights (one scale per output channel): the tokens are
                 quantized to 8 bits (one scale, and in the asymmetric grid one zero point, per
                 token), multiplied with the weights in integers and scaled back
- ``cache``      new keys and values of several sequences written into a paged cache (4 or 8
                 bits, one scale per token and head), then every sequence's last tokens read back
- ``attention``  causal attention of each sequence's new tokens over its keys and values in
                 such a cache: chunks of a prompt, single tokens, or both in one batch

The grid is the framework's: with b bits, codes run from -2^(b-1) to 2^(b-1) - 1; symmetric
``s = max|x| / ((2^b - 1) / 2)``; asymmetric ``s = (max(x, 0) - min(x, 0)) / (2^b - 1)`` and zero
point ``z = clamp(round(minq - min(x, 0) / s))``; ``q = clamp(round(x / s) + z)``, every quotient
rounded to 32 bits and ``round`` half to even.  A code stands for ``s * (q - z)``.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding step of one user: an attention projection of a single token (latency)
        {"name": "linear_token", "op": "linear", "tokens": 1, "rows": 4096, "cols": 4096,
         "sym": True, "bias": False, "dtype": "bf16"},
        # a decoding step of 48 users through the up projection: the weights' bytes count
        {"name": "linear_decode", "op": "linear", "tokens": 48, "rows": 14336, "cols": 4096,
         "sym": True, "bias": False, "dtype": "bf16"},
        # ragged sizes, the asymmetric grid and a bias, fp16 model
        {"name": "linear_ragged", "op": "linear", "tokens": 777, "rows": 1000, "cols": 2752,
         "sym": False, "bias": True, "dtype": "fp16"},
        # a prompt's batch through the up projection: matrix cores
        {"name": "linear_prompt", "op": "linear", "tokens": 8192, "rows": 14336, "cols": 4096,
         "sym": True, "bias": False, "dtype": "bf16"},
        # one decoding step of 32 users: a token each, short tails read back (latency)
        {"name": "cache_token", "op": "cache", "seqs": 32, "new": 1, "tail": 16, "even": True,
         "heads": 8, "dim": 128, "bits": 8, "sym": True, "page": 16, "dtype": "bf16"},
        # prompts of uneven lengths, 4 bits asymmetric, narrow heads, fp16 model
        {"name": "cache_uneven", "op": "cache", "seqs": 11, "new": 600, "tail": 600,
         "even": False, "heads": 4, "dim": 64, "bits": 4, "sym": False, "page": 16,
         "dtype": "fp16"},
        # one long prompt as a calibration run passes it: written and read back whole
        {"name": "cache_prompt", "op": "cache", "seqs": 1, "new": 8192, "tail": 8192,
         "even": True, "heads": 8, "dim": 128, "bits": 4, "sym": False, "page": 64,
         "dtype": "bf16"},
        # a chunk per user on long contexts, the contexts read back
        {"name": "cache_long", "op": "cache", "seqs": 16, "new": 512, "tail": 8192, "even": True,
         "heads": 8, "dim": 128, "bits": 8, "sym": True, "page": 64, "dtype": "bf16"},
        # one user's next token over a context of some thousand tokens (latency)
        {"name": "attend_token", "op": "attention", "seqs": 1, "new": 1, "context": 4001,
         "even": True, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "sym": True,
         "page": 64, "dtype": "bf16"},
        # a decoding step of 64 users with contexts of all lengths, 4-bit cache
        {"name": "attend_decode", "op": "attention", "seqs": 64, "new": 1, "context": 8192,
         "even": False, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 4, "sym": False,
         "page": 64, "dtype": "bf16"},
        # prompts' chunks of uneven lengths, small pages, narrow heads, fp16 model
        {"name": "attend_uneven", "op": "attention", "seqs": 6, "new": 200, "context": 1500,
         "even": False, "heads": 12, "kv_heads": 4, "dim": 64, "bits": 4, "sym": False,
         "page": 16, "dtype": "fp16"},
        # a chunk of a long prompt over what the cache has of it: matrix cores
        {"name": "attend_chunk", "op": "attention", "seqs": 1, "new": 2048, "context": 16384,
         "even": True, "heads": 32, "kv_heads": 8, "dim": 128, "bits": 8, "sym": True,
         "page": 64, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "cache", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "linear":
        tokens, rows, cols = _log(rng, 1, 8192), _log(rng, 256, 14336), _log(rng, 256, 14336)
        while tokens * rows * cols > 8192 * 14336 * 4096:
            tokens = max(1, tokens // 2)
        return {"op": op, "tokens": tokens, "rows": rows, "cols": cols,
                "sym": rng.random() < 0.6, "bias": rng.random() < 0.5,
                "dtype": rng.choice([dtype, dtype, "fp32"])}
    bits, page = rng.choice([4, 8]), rng.choice([16, 32, 64, 128])
    dim = rng.choice([64, 128])
    case = {"op": op, "seqs": _log(rng, 1, 64), "even": rng.random() < 0.3, "dim": dim,
            "bits": bits, "sym": rng.random() < 0.5, "page": page, "dtype": dtype}
    if op == "cache":
        case["heads"] = rng.choice([1, 2, 4, 8])
        case["new"] = _log(rng, 1, max(2, 8192 // case["seqs"]))
        case["tail"] = case["new"] + _log(rng, 1, max(2, 65536 // case["seqs"]))
        return case
    kv = rng.choice([1, 2, 4, 8])
    case["heads"], case["kv_heads"] = kv * rng.choice([1, 3, 4, 8][:3 if kv == 8 else 4]), kv
    case["new"] = rng.choice([1, _log(rng, 2, 2048)])
    case["context"] = case["new"] + _log(rng, 1, 14000)
    while (case["seqs"] * case["new"] * case["context"] > 2048 * 16384
           or case["seqs"] * case["context"] > 64 * 8192):
        case["seqs"] //= 2  # one sequence is within both
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(case):
    """Per sequence: new tokens and tokens in the cache after them (host numbers)."""
    rng = random.Random(1)
    n, new, whole = case["seqs"], case["new"], case.get("context", case.get("tail"))
    if case["even"]:
        return [new] * n, [max(whole, new)] * n
    news, wholes = [], []
    for i in range(n):
        k = new if i == 0 else rng.randint(1, new)
        news.append(k)
        wholes.append(max(whole if i == 0 else rng.randint(1, whole), k))
    return news, wholes


def _keys(g, tokens, heads, dim, dtype):
    """Keys or values: channels of their own sizes, some tokens larger than others."""
    channel = torch.exp(0.5 * torch.randn(heads, dim, generator=g, device=DEV))
    token = torch.exp(0.3 * torch.randn(tokens, 1, 1, generator=g, device=DEV))
    x = torch.randn(tokens, heads, dim, generator=g, device=DEV)
    return x.mul_(channel).mul_(token).add_(0.2).to(dtype)


def _offsets(lengths):
    return torch.tensor([0] + np.cumsum(lengths).tolist(), dtype=torch.int32, device=DEV)


def _inputs(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    if case["op"] == "linear":
        T, N, K = case["tokens"], case["rows"], case["cols"]
        channel = torch.exp(0.5 * torch.randn(K, generator=g, device=DEV))
        x = (torch.randn(T, K, generator=g, device=DEV) * channel).to(dtype)
        codes = torch.randn(N, K, generator=g, device=DEV).mul_(40).round_().clamp_(-128, 127)
        scale = 1e-4 * (0.5 + torch.rand(N, generator=g, device=DEV))
        bias = 0.1 * torch.randn(N, generator=g, device=DEV) if case["bias"] else None
        return {"x": x, "codes": codes.to(torch.int8), "scale": scale, "bias": bias}
    news, wholes = _lengths(case)
    page, D = case["page"], case["dim"]
    H = case["heads"] if case["op"] == "cache" else case["kv_heads"]
    pages = [-(-w // page) for w in wholes]
    total = sum(pages)
    # pages come from a pool in no order; a table row holds its sequence's pages, then zeros
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(news), max(pages), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"table": table, "pages": total, "cu_new": _offsets(news), "cu_whole": _offsets(wholes),
         "lengths": torch.tensor(wholes, dtype=torch.int32, device=DEV), "news": news,
         "wholes": wholes}

    def slots(first, last):  # cache slots of every sequence's tokens first .. last - 1
        seq = torch.cat([torch.full((b - a,), i, dtype=torch.int64) for i, (a, b) in
                         enumerate(zip(first, last))]).to(DEV)
        pos = torch.cat([torch.arange(a, b) for a, b in zip(first, last)]).to(DEV)
        return table[seq, pos // page].long() * page + pos % page

    s["old"] = slots([0] * len(news), [w - n for w, n in zip(wholes, news)])
    s["new"] = slots([w - n for w, n in zip(wholes, news)], wholes)
    s["all"] = slots([0] * len(news), wholes)
    s["k_old"] = _keys(g, s["old"].numel(), H, D, dtype)
    s["v_old"] = _keys(g, s["old"].numel(), H, D, dtype)
    T = s["new"].numel()
    # queries, keys and values are views of one projection's output
    Hq = case["heads"] if case["op"] == "attention" else H
    qkv = torch.cat([_keys(g, T, Hq, D, dtype), _keys(g, T, H, D, dtype),
                     _keys(g, T, H, D, dtype)], dim=1)
    s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["dtype"] = case, DTYPES[case["dtype"]]
    if case["op"] == "linear":
        if own:
            from g2ptq_amd import Int8Linear
            s["linear"] = Int8Linear(s["codes"], s["scale"], bias=s["bias"], sym=case["sym"])
        return s
    H, s["max_q"], s["max_kv"] = s["k"].shape[1], max(s["news"]), max(s["wholes"])
    if own:
        from g2ptq_amd import PagedKVCache
        s["cache"] = PagedKVCache(s["pages"], case["page"], H, case["dim"], bits=case["bits"],
                                  sym=case["sym"], device=DEV)
        s["cache"].write(s["k_old"], s["v_old"], s["old"])
        if case["op"] == "attention":
            s["cache"].write(s["k"], s["v"], s["new"])
    else:
        # per slot and head: codes, scale and zero point of keys and of values
        n = s["pages"] * case["page"]
        s["codes"] = torch.zeros(2, n, H, case["dim"], device=DEV)
        s["scale"], s["zero"] = torch.zeros(2, 2, n, H, 1, device=DEV)
        _plain_write(s, s["k_old"], s["v_old"], s["old"])
        if case["op"] == "attention":
            _plain_write(s, s["k"], s["v"], s["new"])
    return s


# ---------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_quantize(x, bits, sym):
    """Codes, scale and zero point of the grid above along the last axis."""
    x = x.float()
    minq, maxq = -(1 << (bits - 1)), (1 << (bits - 1)) - 1
    zero = torch.zeros(x.shape[:-1] + (1,), device=x.device)
    if sym:
        half = torch.full_like(zero, (maxq - minq) / 2)
        scale = x.abs().amax(-1, keepdim=True) / half
    else:
        lo = x.amin(-1, keepdim=True).clamp(max=0)
        hi = x.amax(-1, keepdim=True).clamp(min=0)
        scale = (hi - lo) / torch.full_like(zero, maxq - minq)
        zero = (minq - lo / scale).round().clamp(minq, maxq)
    q = ((x / scale).round() + zero).clamp(minq, maxq)
    flat = scale == 0  # nothing but zeros: code and zero point 0
    return torch.where(flat, 0.0, q), scale, torch.where(flat, 0.0, zero)


def _plain_write(s, k, v, slots):
    new = _plain_quantize(torch.stack([k, v]), s["case"]["bits"], s["case"]["sym"])
    s["codes"][:, slots], s["scale"][:, slots], s["zero"][:, slots] = new


def _plain_read(s, slots):
    return s["scale"][:, slots] * (s["codes"][:, slots] - s["zero"][:, slots])


def _plain_attention(s):
    """Every sequence padded to the most new tokens and the longest context of the batch."""
    case, table, cu, lengths = s["case"], s["table"], s["cu_new"].long(), s["lengths"].long()
    Hq, H, D, B, T = case["heads"], case["kv_heads"], case["dim"], table.shape[0], len(s["q"])
    token = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu[1:], token, right=True)
    at = token - cu[seq]
    q = torch.zeros(B, s["max_q"], Hq, D, device=DEV)
    q[seq, at] = s["q"].float()
    q = q.permute(0, 2, 1, 3).reshape(B, H, Hq // H * s["max_q"], D)
    key = torch.arange(s["max_kv"], device=DEV)
    k, v = _plain_read(s, table[:, key // case["page"]].long() * case["page"] + key % case["page"])
    logits = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(D))
    logits = logits.view(B, Hq, s["max_q"], -1)
    # a query sees the keys up to its own; rows that pad the batch see the first key
    last = (lengths - cu.diff()).unsqueeze(1) + torch.arange(s["max_q"], device=DEV)
    seen = key <= last[:, None, :, None]
    p = torch.where(seen, logits, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, H, Hq // H * s["max_q"], -1)
    o = torch.matmul(p, v.transpose(1, 2).contiguous()).view(B, Hq, s["max_q"], D)
    return o[seq, :, at].to(s["dtype"])


def run(s):
    case = s["case"]
    if own:
        if case["op"] == "linear":
            return s["linear"](s["x"])
        if case["op"] == "cache":
            s["cache"].write(s["k"], s["v"], s["new"])
            return s["cache"].read(s["table"], s["cu_whole"], s["all"].numel(), dtype=s["dtype"])
        from g2ptq_amd import paged_attention
        return paged_attention(s["q"], s["cache"], s["table"], s["cu_new"], s["lengths"],
                               max_q=s["max_q"], max_kv=s["max_kv"])
    if case["op"] == "linear":
        q, scale, zero = _plain_quantize(s["x"], 8, case["sym"])
        w = s["codes"].float()
        y = torch.matmul(q, w.t()) - zero * w.sum(-1)
        y = y * scale * s["scale"]
        return (y if s["bias"] is None else y + s["bias"]).to(s["dtype"])
    if case["op"] == "cache":
        _plain_write(s, s["k"], s["v"], s["new"])
        k, v = _plain_read(s, s["all"]).to(s["dtype"])
        return [k, v]
    return _plain_attention(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "linear":
        T, N, K = case["tokens"], case["rows"], case["cols"]
        return {"bytes": T * K * e + N * K + N * (8 if case["bias"] else 4) + T * N * e,
                "flops": 2 * T * N * K}
    H = case["heads"] if case["op"] == "cache" else case["kv_heads"]
    news, wholes = _lengths(case)
    held = 2 * H * (case["dim"] * case["bits"] / 8 + (4 if case["sym"] else 5))
    plain = 2 * H * case["dim"] * e
    new, whole = sum(news), sum(wholes)
    if case["op"] == "cache":
        return {"bytes": int(new * (plain + held) + whole * (held + plain)),
                "flops": int((new + whole) * 2 * H * case["dim"] * 4)}
    pairs = sum(n * (w - n) + n * (n + 1) // 2 for n, w in zip(news, wholes))
    return {"bytes": int(whole * held + 2 * new * case["heads"] * case["dim"] * e),
            "flops": 4 * case["heads"] * case["dim"] * pairs}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_grid(x, bits, sym):
    """(codes - zero, scale) along the last axis; numbers that the definition rounds to 32 bits
    (scales, quotients) are computed in 64 and rounded."""
    x = x.double()
    top, lowest = 2.0 ** (bits - 1) - 1, -2.0 ** (bits - 1)

    def divided(a, b):  # a / b rounded to 32 bits; 0 / 0 counts as 0
        r = torch.where(b == 0, torch.zeros_like(a), a / torch.where(b == 0, 1.0, b))
        return r.float().double()

    if sym:
        s = (torch.max(x.abs(), dim=-1, keepdim=True)[0] / (top + 0.5)).float().double()
        return torch.clamp(torch.round(divided(x, s)), lowest, top), s
    low = torch.min(x, dim=-1, keepdim=True)[0].clamp(max=0)
    high = torch.max(x, dim=-1, keepdim=True)[0].clamp(min=0)
    s = ((high - low).float().double() / (2 * top + 1)).float().double()
    z = torch.clamp(torch.round((lowest - divided(low, s)).float().double()), lowest, top)
    z = torch.where(s == 0, torch.zeros_like(z), z)
    return torch.clamp(torch.round(divided(x, s)) + z, lowest, top) - z, s


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        c, scale = _exact_grid(s["x"], 8, case["sym"])
        y = (c @ s["codes"].double().t()) * (scale * s["scale"].double())
        return y if s["bias"] is None else y + s["bias"].double()
    held = []
    for old, new in ((s["k_old"], s["k"]), (s["v_old"], s["v"])):
        c, scale = _exact_grid(torch.cat([old, new]), case["bits"], case["sym"])
        x = torch.zeros(s["pages"] * case["page"], *new.shape[1:], dtype=torch.float64, device=DEV)
        x[torch.cat([s["old"], s["new"]])] = c * scale
        held.append(x[s["all"]])
    if case["op"] == "cache":
        return held
    k, v = held
    share = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    start, first = 0, 0
    for n, w in zip(s["news"], s["wholes"]):
        ahead = torch.ones(n, w, dtype=torch.bool, device=DEV).triu(w - n + 1)
        for h in range(case["heads"]):
            kh, vh = k[first:first + w, h // share], v[first:first + w, h // share]
            logits = s["q"][start:start + n, h].double() @ kh.t().contiguous() / case["dim"] ** 0.5
            logits = logits.masked_fill(ahead, -math.inf)
            out[start:start + n, h] = torch.softmax(logits, dim=-1) @ vh
        start, first = start + n, first + w
    return out
