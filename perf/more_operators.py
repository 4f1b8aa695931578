"""Performance cases of the operators that stand between the products of a served quantized layer.

``op`` of a case:

- ``norm``      root-mean-square norm of every row, with the residual's addition where there is
                one: ``s = x + r``, ``y = s * w / sqrt(mean(s^2) + eps)``; ``y`` comes in the
                inputs' type, or quantized to 8 bits (one scale, and in the asymmetric grid one
                zero point, per row) and returned as the values that the codes stand for
- ``rotary``    rotary positions of queries and keys: pair i of a token's head is turned by
                ``position * f_i``; pairs are channels (i, i + n/2) or (2i, 2i + 1) of the first n
- ``pages``     a batch's requests get new tokens in a paged cache: pages from a stack of free
                ones, the batch's page tables, every token's slot and position; then the tokens
                are taken back (a draft that is not kept), which restores the stack
- ``adapters``  low-rank adapters of many requests beside a shared projection: to each token's
                row of the projection's output its own adapter's part is added

The 8-bit grid is the framework's: symmetric ``s = max|y| / 127.5``; asymmetric
``s = (max(y, 0) - min(y, 0)) / 255`` and ``z = clamp(round(-128 - min(y, 0) / s))``;
``q = clamp(round(y / s) + z)``.  A code stands for ``s * (q - z)``.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def listed():
    return [
        # one decoding step of one user: the norm before a layer's projections (latency)
        {"name": "norm_token", "op": "norm", "tokens": 1, "heads": 1, "cols": 4096,
         "residual": True, "quantize": True, "sym": True, "dtype": "bf16"},
        # ragged sizes, the residual's stream in fp16, output in the type
        {"name": "norm_ragged", "op": "norm", "tokens": 777, "heads": 1, "cols": 2752,
         "residual": True, "quantize": False, "sym": True, "dtype": "fp16"},
        # the norm of every head of a prompt's queries, which are a view of the projections
        {"name": "norm_heads", "op": "norm", "tokens": 8192, "heads": 32, "cols": 128,
         "residual": False, "quantize": False, "sym": True, "dtype": "bf16"},
        # a prompt's batch before the projections of a layer
        {"name": "norm_prompt", "op": "norm", "tokens": 8192, "heads": 1, "cols": 4096,
         "residual": True, "quantize": True, "sym": True, "dtype": "bf16"},
        # one user's next token far into a long context (latency)
        {"name": "rotary_token", "op": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "part": 128, "layout": "half", "scaling": "none", "far": 100000,
         "dtype": "bf16"},
        # prompts of a fp16 model that turns half of a head, in neighbouring pairs
        {"name": "rotary_ragged", "op": "rotary", "tokens": 777, "heads": 12, "kv_heads": 4,
         "dim": 64, "part": 32, "layout": "interleaved", "scaling": "yarn", "far": 30000,
         "dtype": "fp16"},
        # a chunk of long prompts, frequencies scaled for long contexts
        {"name": "rotary_prompt", "op": "rotary", "tokens": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "part": 128, "layout": "half", "scaling": "bands", "far": 131072,
         "dtype": "bf16"},
        # one decoding step of 32 users: a token each (latency)
        {"name": "pages_token", "op": "pages", "seqs": 32, "new": 1, "held": 2000, "even": True,
         "page": 16},
        # chunks of many users' prompts, of uneven lengths, behind what the cache has of them
        {"name": "pages_prompt", "op": "pages", "seqs": 700, "new": 2048, "held": 6000,
         "even": False, "page": 64},
        # a decoding step of 48 users with 32 adapters through an attention projection
        {"name": "adapters_token", "op": "adapters", "seqs": 48, "new": 1, "adapters": 32,
         "rank": 16, "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # chunks of uneven prompts, ragged sizes, adapters of several ranks, fp16 model
        {"name": "adapters_uneven", "op": "adapters", "seqs": 9, "new": 200, "adapters": 5,
         "rank": 24, "rows": 1000, "cols": 2752, "dtype": "fp16"},
        # a batch of prompts through the up projection
        {"name": "adapters_prompt", "op": "adapters", "seqs": 8, "new": 1024, "adapters": 4,
         "rank": 64, "rows": 14336, "cols": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "pages", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        if rng.random() < 0.3:  # heads
            case = {"tokens": _log(rng, 1, 8192), "heads": rng.choice([1, 4, 8, 32]),
                    "cols": rng.choice([64, 96, 128, 256]), "residual": False, "quantize": False}
        else:
            case = {"tokens": _log(rng, 1, 8192), "heads": 1, "cols": _log(rng, 256, 16384),
                    "residual": rng.random() < 0.7, "quantize": rng.random() < 0.6}
            while case["tokens"] * case["cols"] > 8192 * 4096:
                case["tokens"] = max(1, case["tokens"] // 2)
        if not case["quantize"]:
            dtype = rng.choice([dtype, dtype, "fp32"])
        return {"op": op, **case, "sym": rng.random() < 0.6, "dtype": dtype}
    if op == "rotary":
        dim = rng.choice([64, 80, 128, 192])
        kv = rng.choice([1, 2, 4, 8])
        case = {"op": op, "tokens": _log(rng, 1, 16384), "heads": kv * rng.choice([1, 3, 4]),
                "kv_heads": kv, "dim": dim,
                "part": rng.choice([dim, dim, dim // 2, max(2, dim // 4 // 2 * 2)]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                "far": _log(rng, 100, 1000000), "dtype": dtype}
        while case["tokens"] * (case["heads"] + kv) * dim > 16384 * 40 * 128:
            case["tokens"] //= 2
        return case
    if op == "pages":
        case = {"op": op, "seqs": _log(rng, 1, 1000), "new": rng.choice([1, _log(rng, 2, 2048)]),
                "held": _log(rng, 1, 6000), "even": rng.random() < 0.3,
                "page": rng.choice([16, 32, 64, 128])}
        while (case["seqs"] * case["new"] > 700 * 1024
               or case["seqs"] * (case["new"] + case["held"]) // case["page"] > 88000):
            case["seqs"] //= 2
        return case
    case = {"op": op, "seqs": _log(rng, 1, 64), "new": rng.choice([1, _log(rng, 2, 2048)]),
            "adapters": _log(rng, 1, 40), "rank": rng.choice([8, 16, 16, 24, 32, 64]),
            "rows": _log(rng, 256, 14336), "cols": _log(rng, 256, 14336), "dtype": dtype}
    while (case["seqs"] * case["new"] * (case["rows"] + case["cols"]) > 8192 * 18432
           or case["adapters"] * case["rank"] * (case["rows"] + case["cols"])
           * max(16, case["seqs"] * case["new"] // 8) > 256 * 18432 * 1024):
        if case["seqs"] > 1:
            case["seqs"] //= 2
        elif case["new"] > 1:
            case["new"] //= 2
        else:
            case["adapters"] = max(1, case["adapters"] // 2)
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _counts(case, seqs, most):
    """Per request: a host number from 1 to ``most`` (the first has all)."""
    rng = random.Random(1)
    return [most if case.get("even") or i == 0 else rng.randint(1, most) for i in range(seqs)]


def _ranks(case):
    """Where there are several adapters, some have half the rank."""
    return [max(1, case["rank"] // 2) if i % 3 == 1 else case["rank"]
            for i in range(case["adapters"])]


def _activations(g, *shape, dtype):
    """Rows of their own sizes, channels of their own sizes, a few channels far above."""
    channel = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    channel = torch.where(torch.rand(shape[-1], generator=g, device=DEV) < 0.004, 20.0, channel)
    row = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g, device=DEV))
    return (torch.randn(*shape, generator=g, device=DEV) * channel * row).to(dtype)


def _frequencies(case):
    """Radians a position turns pair i by (64 bits), and the factor on cosine and sine."""
    n, base, factor, trained = case["part"], 500000.0, 8.0, 8192.0
    i = torch.arange(0, n, 2, dtype=torch.float64) / n
    if case["scaling"] == "ntk" and n > 2:
        base *= factor ** (n / (n - 2))
    f = base ** -i
    turns = trained * f / (2 * math.pi)  # over the trained length
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":
        # pairs between those that turn 32 times and once over the trained length: a ramp
        first, last = (n * math.log(trained / (k * 2 * math.pi)) / (2 * math.log(base))
                       for k in (32.0, 1.0))
        first, last = max(math.floor(first), 0), min(math.ceil(last), n - 1)
        ramp = ((torch.arange(n // 2, dtype=torch.float64) - first)
                / max(last - first, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if case["scaling"] == "bands":
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f / factor * (1 - smooth) + f * smooth
    return f, 1.0


def _scaling(case):
    """The same for the framework."""
    return {"none": None, "linear": {"type": "linear", "factor": 8.0},
            "ntk": {"type": "ntk", "factor": 8.0},
            "yarn": {"type": "yarn", "factor": 8.0, "original_positions": 8192},
            "bands": {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0,
                      "high_freq_factor": 4.0, "original_positions": 8192}}[case["scaling"]]


def _inputs(case, seed):
    g, dtype = _generator(seed), DTYPES.get(case.get("dtype"))
    if case["op"] == "norm":
        T, H, C = case["tokens"], case["heads"], case["cols"]
        s = {"w": (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(dtype), "r": None}
        if H > 1:  # the queries' part of the projections' output
            s["x"] = _activations(g, T, H + 16, C, dtype=dtype)[:, :H]
        else:
            s["x"] = _activations(g, T, C, dtype=dtype)
        if case["residual"]:
            s["r"] = _activations(g, T, C, dtype=dtype)
        return s
    if case["op"] == "rotary":
        T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = _activations(g, T, H + 2 * K, D, dtype=dtype)  # one projection's output
        # chunks of up to 4096 tokens, each somewhere in its context
        chunk = torch.arange(T, device=DEV) // 4096
        start = torch.randint(0, case["far"], (T // 4096 + 1,), generator=g, device=DEV)
        return {"q": qkv[:, :H], "k": qkv[:, H:H + K],
                "positions": start[chunk] + torch.arange(T, device=DEV) % 4096}
    B, new = case["seqs"], _counts(case, case["seqs"], case["new"])
    if case["op"] == "pages":
        held = _counts(case, B, case["held"])[::-1]
        spare = B // 8 + 16  # requests that are not in this batch
        pages = sum(-(-(n + h) // case["page"]) for n, h in zip(new, held))
        order = torch.randperm(B + spare, generator=g, device=DEV).to(torch.int32)
        return {"rows": order[:B].contiguous(), "others": order[B:].contiguous(),
                "seqs": B + spare, "total": sum(new),
                "pages": pages + (spare * case["held"]) // case["page"] + 2 * spare,
                "width": max(-(-(n + h) // case["page"]) for n, h in zip(new, held)) + 3,
                "new": torch.tensor(new, dtype=torch.int32, device=DEV),
                "held": torch.tensor(held, dtype=torch.int32, device=DEV)}
    T, n, r, N, K = sum(new), case["adapters"], case["rank"], case["rows"], case["cols"]
    ranks = _ranks(case)
    of = torch.randint(-1 if n > 2 else 0, n, (B,), generator=g, device=DEV)
    s = {"x": _activations(g, T, K, dtype=dtype),
         "base": torch.randn(T, N, generator=g, device=DEV).to(dtype),
         "index": torch.repeat_interleave(of, torch.tensor(new, device=DEV)).to(torch.int32),
         "down": [(torch.randn(k, K, generator=g, device=DEV) / math.sqrt(K)).to(dtype)
                  for k in ranks],
         "up": [(torch.randn(N, k, generator=g, device=DEV) / math.sqrt(k)).to(dtype)
                for k in ranks],
         "scale": [0.5 + 0.25 * (i % 4) for i in range(n)]}
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["dtype"] = case, DTYPES.get(case.get("dtype"))
    if case["op"] == "rotary":
        if own:
            from g2ptq_amd import Rotary
            s["rotary"] = Rotary(case["dim"], rotary_dim=case["part"], base=500000.0,
                                 layout=case["layout"], scaling=_scaling(case), device=DEV)
        else:
            s["frequencies"], s["factor"] = _frequencies(case)
            s["frequencies"] = s["frequencies"].to(DEV)
    if case["op"] == "pages":
        if own:
            from g2ptq_amd import PageTables
            s["tables"] = PageTables(s["pages"], case["page"], s["seqs"], s["width"], device=DEV)
        else:
            # stack of free pages (the last on top), pages of every request, its tokens
            s["free"] = torch.arange(s["pages"] - 1, -1, -1, dtype=torch.int32, device=DEV)
            s["count"] = torch.tensor([s["pages"]], dtype=torch.int32, device=DEV)
            s["table"] = torch.full((s["seqs"], s["width"]), -1, dtype=torch.int32, device=DEV)
            s["lengths"] = torch.zeros(s["seqs"], dtype=torch.int32, device=DEV)
        # the batch's requests came in two steps, others came and went
        half = s["held"] // 2
        some = torch.full_like(s["others"], min(case["held"], s["width"] * case["page"]))
        for rows, new in ((s["rows"], half), (s["others"], some), (s["rows"], s["held"] - half)):
            _extend(s, rows, new, int(new.sum()))
        _release(s, s["others"][::2].contiguous(), None)
    if case["op"] == "adapters" and own:
        from g2ptq_amd import LowRankAdapters
        s["adapters"] = LowRankAdapters(s["down"], s["up"], scale=s["scale"])
    elif case["op"] == "adapters":
        # all of one rank, zeros behind the smaller ones
        r = case["rank"]
        s["down"] = torch.stack([torch.nn.functional.pad(d, (0, 0, 0, r - d.shape[0]))
                                 for d in s["down"]])
        s["up"] = torch.stack([torch.nn.functional.pad(u, (0, r - u.shape[1])) for u in s["up"]])
        s["scale"] = torch.tensor(s["scale"], device=DEV)
    return s


# ---------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_norm(s):
    case, dtype = s["case"], s["dtype"]
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    out = {"y": y}
    if case["quantize"]:
        zero = torch.zeros(y.shape[:-1] + (1,), device=DEV)
        if case["sym"]:
            scale = y.abs().amax(-1, keepdim=True) / 127.5
        else:
            low, high = y.amin(-1, keepdim=True).clamp(max=0), y.amax(-1, keepdim=True).clamp(min=0)
            scale = (high - low) / 255
            zero = (-128 - low / scale).round().clamp(-128, 127)
        q = ((y / scale).round() + zero).clamp(-128, 127)
        out["y"], out["scale"] = scale * (q - zero), scale.squeeze(-1)
    out["y"] = out["y"].to(dtype)
    if s["r"] is not None:
        out["sum"] = h.to(dtype)
    return out


def _plain_rotary(s, x):
    case, n = s["case"], s["case"]["part"]
    angle = torch.remainder(s["positions"].double().unsqueeze(1) * s["frequencies"], 2 * math.pi)
    c, si = ((f(angle) * s["factor"]).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    x = x.float()
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * c - b * si, a * si + b * c], -1)
    else:
        a, b = x[..., :n:2], x[..., 1:n:2]
        turned = torch.stack([a * c - b * si, a * si + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1).to(s["dtype"])


def _extend(s, rows, new, total):
    """Pages, slots and positions of the requests' new tokens."""
    page = s["case"]["page"]
    if own:
        return s["tables"].extend(rows, new, total)
    at, width = rows.long(), s["width"]
    before = s["lengths"][at]
    after = before + new
    had, need = -(-before // page), -(-after // page)
    # pages come from the top of the stack, request by request
    cum = torch.cumsum(need - had, 0)
    top = s["count"] - 1 - (cum - (need - had))
    column = torch.arange(width, device=DEV)
    fresh = (column >= had.unsqueeze(1)) & (column < need.unsqueeze(1))
    place = (top + had).unsqueeze(1) - column
    table = torch.where(fresh, s["free"][place.clamp(0, s["pages"] - 1)], s["table"][at])
    s["table"][at] = table
    s["lengths"][at] = after
    s["count"] -= cum[-1:].to(torch.int32)
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0).to(torch.int32)])
    token = torch.arange(total, device=DEV)
    seq = torch.searchsorted(cu[1:].long(), token, right=True)
    position = before[seq].long() + token - cu[seq].long()
    slots = table[seq, position // page].long() * page + position % page
    return table, cu, after, slots, position


def _release(s, rows, keep):
    """The requests' pages back onto the stack, the first of them on top."""
    if own:
        return s["tables"].release(rows, keep)
    page, at = s["case"]["page"], rows.long()
    keep = torch.zeros_like(rows) if keep is None else keep
    kept, had = -(-keep // page), -(-s["lengths"][at] // page)
    column = torch.arange(s["width"], device=DEV)
    gone = (column >= kept.unsqueeze(1)) & (column < had.unsqueeze(1))
    cum = torch.cumsum(had - kept, 0)
    order = (cum - (had - kept)).unsqueeze(1) + column - kept.unsqueeze(1)
    # (pages that stay go nowhere: one place behind the stack)
    place = torch.where(gone, s["count"] + cum[-1] - 1 - order, s["pages"]).long()
    free = torch.cat([s["free"], s["free"][:1]])
    free[place] = s["table"][at]
    s["free"] = free[:-1]
    s["table"][at] = torch.where(gone, -1, s["table"][at])
    s["lengths"][at] = keep
    s["count"] += cum[-1:].to(torch.int32)


def _plain_adapters(s):
    """Every token through every adapter, all but its own masked out."""
    n = s["down"].shape[0]
    h = torch.matmul(s["x"].float(), s["down"].float().flatten(0, 1).t())
    mine = s["index"].unsqueeze(1) == torch.arange(n, device=DEV)
    h = h.view(-1, n, s["case"]["rank"]) * (mine * s["scale"]).unsqueeze(-1)
    up = s["up"].float().transpose(1, 2).flatten(0, 1)
    return (s["base"].float() + torch.matmul(h.flatten(1), up)).to(s["dtype"])


def run(s):
    case = s["case"]
    if case["op"] == "norm":
        if not own:
            return _plain_norm(s)
        from g2ptq_amd import dequantize_tokens, rms_norm, rms_norm_quantize
        if not case["quantize"]:
            y = rms_norm(s["x"], s["w"], EPS, residual=s["r"])
            return {"y": y} if s["r"] is None else {"y": y[0], "sum": y[1]}
        t = rms_norm_quantize(s["x"], s["w"], EPS, residual=s["r"], sym=case["sym"])
        out = {"y": dequantize_tokens(t.codes, t.scale, t.zero, dtype=s["dtype"]),
               "scale": t.scale}
        if s["r"] is not None:
            out["sum"] = t.sum
        return out
    if case["op"] == "rotary":
        if own:
            return list(s["rotary"](s["q"], s["k"], s["positions"]))
        return [_plain_rotary(s, s["q"]), _plain_rotary(s, s["k"])]
    if case["op"] == "pages":
        step = list(_extend(s, s["rows"], s["new"], s["total"]))
        _release(s, s["rows"], s["held"])
        state = s["tables"] if own else None
        if own:
            return step + [state.table, state.lengths, state.free_pages, state.free_count]
        return step + [s["table"], s["lengths"], s["free"], s["count"]]
    if own:
        return s["adapters"](s["x"], s["index"], base=s["base"])
    return _plain_adapters(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = SIZE.get(case.get("dtype"))
    if case["op"] == "norm":
        rows, C = case["tokens"] * case["heads"], case["cols"]
        moved = 2 + 2 * case["residual"]  # x and y, the residual and the sum
        scales = rows * (4 if case["sym"] else 8) if case["quantize"] else 0
        return {"bytes": moved * rows * C * e + C * e + scales,
                "flops": rows * C * (4 + case["residual"] + 4 * case["quantize"])}
    if case["op"] == "rotary":
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": case["tokens"] * (2 * heads * case["dim"] * e + 8),
                "flops": case["tokens"] * heads * case["part"] * 3}
    new = _counts(case, case["seqs"], case["new"])
    if case["op"] == "pages":
        held = _counts(case, case["seqs"], case["held"])[::-1]
        pages = [-(-(n + h) // case["page"]) for n, h in zip(new, held)]
        # the batch's tables and what they are made of; slots and positions; counts and offsets
        return {"bytes": 4 * (case["seqs"] * (max(pages) + 3) + sum(pages)) + 16 * sum(new)
                + 28 * case["seqs"], "flops": 4 * sum(new)}
    T, N, K = sum(new), case["rows"], case["cols"]
    n = case["adapters"]
    rank = sum(_ranks(case)) / n  # of the requests' adapters, on average
    return {"bytes": int(e * (T * (K + 2 * N) + min(n, case["seqs"]) * rank * (K + N))) + 4 * T,
            "flops": int(2 * T * rank * (K + N))}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(case, s):
    h = s["x"].double() if s["r"] is None else s["x"].double() + s["r"].double()
    size = (h * h).sum(-1, keepdim=True) / case["cols"] + EPS
    y = s["w"].double() * h * size.rsqrt()
    out = {"y": y}
    if s["r"] is not None:
        out["sum"] = h
    if case["quantize"]:
        if case["sym"]:
            scale, zero = torch.max(y.abs(), -1, keepdim=True)[0] / 127.5, torch.zeros(1, device=DEV)
        else:
            low = torch.min(y, -1, keepdim=True)[0].clamp(max=0)
            scale = (torch.max(y, -1, keepdim=True)[0].clamp(min=0) - low) / 255
            zero = torch.clamp(torch.round(-128 - low / scale), -128, 127)
        out["y"] = (torch.clamp(torch.round(y / scale) + zero, -128, 127) - zero) * scale
        out["scale"] = scale[..., 0]
    return out


def _exact_rotary(case, s, x):
    f, factor = _frequencies(case)
    angle = s["positions"].double()[:, None] * f.to(DEV)[None]
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    n, x = case["part"], x.double()
    if case["layout"] == "half":
        z = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., n:]], dim=-1)
    z = torch.view_as_complex(x[..., :n].reshape(*x.shape[:-1], n // 2, 2).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).reshape(*x.shape[:-1], n), x[..., n:]], dim=-1)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers
    s = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"] == "rotary":
        return [_exact_rotary(case, s, s["q"]), _exact_rotary(case, s, s["k"])]
    y = s["base"].double()
    for i, (down, up) in enumerate(zip(s["down"], s["up"])):
        t = (s["index"] == i).nonzero()[:, 0]
        h = s["x"][t].double() @ down.double().t().contiguous()
        y[t] += s["scale"][i] * (h @ up.double().t().contiguous())
    return y
