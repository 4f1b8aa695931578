"""Rotary positions of queries and keys.

Pair i of a head's first ``rotary_dim`` channels is turned by ``position · θ_i``,
``θ_i = base^(−2i/rotary_dim)``, or what ``scaling`` makes of it for contexts longer than the
``original_positions`` L that a model was trained on.  With factor s:

- ``linear``  θ / s
- ``ntk``     the same formula with ``base · s^(d/(d − 2))``, d = ``rotary_dim``
- ``yarn``    θ/s and θ mixed by a ramp over the pairs, from the pair that turns ``beta_fast``
              times over L positions (θ up to it) to the one that turns ``beta_slow`` times (θ/s
              from it on), both rounded outward; sine and cosine are multiplied with
              ``attention_factor`` (0.1 · ln s + 1 by default)
- ``bands``   θ where a pair turns more than ``high_freq_factor`` times over L positions, θ/s
              where it turns less than ``low_freq_factor`` times, between them mixed linearly in
              the number of turns

Inference only: nothing here has a gradient.
"""
import math

import torch

from . import _lib
from .int8_utils import _DTYPE_CODE

_CONTIGUOUS = torch.contiguous_format
_FIELDS = {"linear": {"factor"}, "ntk": {"factor"},
           "yarn": {"factor", "original_positions", "beta_fast", "beta_slow", "attention_factor"},
           "bands": {"factor", "original_positions", "low_freq_factor", "high_freq_factor"}}
_OPTIONAL = {"beta_fast", "beta_slow", "attention_factor"}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """``(θ, m)``: radians a position for each pair (fp64, on the CPU) and the factor on sine
    and cosine.  ``scaling``: None or a dict of ``type`` and its fields (see the module)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary positions turn an even number of channels, not {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError(f"rotary positions: base {base}")
    kind = None if scaling is None else scaling.get("type")
    if scaling is not None:
        if kind not in _FIELDS:
            raise ValueError(f"rotary scaling of type {kind!r} (one of {sorted(_FIELDS)})")
        given = set(scaling) - {"type"}
        if given - _FIELDS[kind] or _FIELDS[kind] - _OPTIONAL - given:
            raise ValueError(f"rotary scaling {kind!r} takes {sorted(_FIELDS[kind])}, got "
                             f"{sorted(given)}")
        s = float(scaling["factor"])
        if not (s > 0 and math.isfinite(s)):
            raise ValueError(f"rotary scaling: factor {s}")
    d = rotary_dim
    if kind == "ntk" and d > 2:
        base = base * s ** (d / (d - 2))
    pair = torch.arange(d // 2, dtype=torch.float64, device="cpu")
    theta = float(base) ** (-2 * pair / d)
    if kind == "linear":
        return theta / s, 1.0
    if kind == "yarn":
        L = float(scaling["original_positions"])
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not (L > 0 and fast > slow > 0 and base > 1):
            raise ValueError(f"rotary scaling: {scaling}")
        # the (fractional) pair that turns k times over L positions
        low, high = (d * math.log(L / (2 * math.pi * k)) / (2 * math.log(base))
                     for k in (fast, slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), d - 1)
        ramp = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        m = scaling.get("attention_factor")
        m = (0.1 * math.log(s) + 1.0 if s > 1 else 1.0) if m is None else float(m)
        return theta * (1 - ramp) + theta / s * ramp, m
    if kind == "bands":
        L = float(scaling["original_positions"])
        few, many = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not (L > 0 and many > few):
            raise ValueError(f"rotary scaling: {scaling}")
        mix = ((theta * (L / (2 * math.pi)) - few) / (many - few)).clamp(0, 1)
        return theta * mix + theta / s * (1 - mix), 1.0
    return theta, 1.0


class Rotary:
    """``q, k = rotary(q, k, positions)``.

    ``layout`` "half": channel i is paired with i + rotary_dim/2; "interleaved": 2i with 2i + 1.
    Channels from ``rotary_dim`` (default: all) on stay as they are.  ``frequencies`` (rotary_dim
    / 2 radians a position, numbers or a tensor of any type) and ``attention_factor`` take the place of ``base``
    and ``scaling``.  Nothing is tabulated: angles are fp64 products less their whole turns, off by
    some 2^-52 of position · θ, so that positions are not limited (up to 2^28 the fp32 sine and
    cosine round more), and negative ones turn back."""

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout="half", scaling=None,
                 frequencies=None, attention_factor=None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ("half", "interleaved"):
            raise ValueError(f"Rotary: layout {layout!r} (\"half\" or \"interleaved\")")
        if not 2 <= rotary_dim <= head_dim <= 1024 or rotary_dim % 2:
            raise ValueError(f"Rotary turns an even number of at most 1024 channels, not "
                             f"{rotary_dim} of {head_dim}")
        if frequencies is None:
            theta, factor = rotary_frequencies(rotary_dim, base, scaling)
        else:
            theta = torch.as_tensor(frequencies, dtype=torch.float64).detach().cpu()
            factor = 1.0
            if scaling is not None or tuple(theta.shape) != (rotary_dim // 2,):
                raise ValueError(f"Rotary: frequencies of shape {tuple(theta.shape)}, expected "
                                 f"({rotary_dim // 2},) and no scaling")
        if torch.device(device).type != "cuda":
            raise RuntimeError("Rotary runs on the GPU")
        self.head_dim, self.rotary_dim, self.layout = head_dim, rotary_dim, layout
        self.factor = float(factor if attention_factor is None else attention_factor)
        self.frequencies = theta.contiguous()
        self._turns = (theta / (2 * math.pi)).contiguous().to(device)
        self.device = self._turns.device
        self._device, self._interleaved = self.device.index, layout == "interleaved"

    def __call__(self, q, k, positions):
        """``q`` (tokens, heads, head_dim) and ``k`` (tokens, kv_heads, head_dim; or None), of
        one type (bf16, fp16 or fp32), any strides of token and head, turned by ``positions``
        (tokens,) int64: new contiguous tensors."""
        dim, here, T = self.head_dim, self._device, positions.shape[0] if positions.dim() else 0
        # what is usual passes in one go (a call is a few microseconds); the rest is told apart
        if not (k is not None and q.dim() == k.dim() == 3 and positions.dim() == 1
                and q.shape[0] == k.shape[0] == T and q.shape[2] == k.shape[2] == dim
                and q.stride(2) == k.stride(2) == 1 and q.dtype is k.dtype
                and q.dtype in _DTYPE_CODE and positions.dtype is torch.int64
                and positions.is_contiguous()
                and q.get_device() == k.get_device() == positions.get_device() == here
                and torch._C._cuda_getDevice() == here
                and not q.requires_grad and not k.requires_grad
                and _lib.forward_ad._current_level < 0):
            q, k, positions = self._checked(q, k, positions)
        T = q.shape[0]
        q_out = torch.empty_like(q, memory_format=_CONTIGUOUS)
        k_out = None if k is None else torch.empty_like(k, memory_format=_CONTIGUOUS)
        if T:
            (qt, qh, _), (kt, kh, _) = q.stride(), (0, 0, 0) if k is None else k.stride()
            _lib.call_fast("rotary", _lib.current_stream(), q.data_ptr(), qt, qh, q.shape[1],
                           None if k is None else k.data_ptr(), kt, kh,
                           0 if k is None else k.shape[1], _DTYPE_CODE[q.dtype], T, dim,
                           self.rotary_dim, self._interleaved, positions.data_ptr(),
                           self._turns.data_ptr(), self.factor, q_out.data_ptr(),
                           None if k is None else k_out.data_ptr())
        return q_out, k_out

    def _checked(self, q, k, positions):
        dim = self.head_dim
        if positions.dtype is not torch.int64 or positions.dim() != 1:
            raise ValueError(f"Rotary: positions of {positions.dtype} and shape "
                             f"{tuple(positions.shape)} (int64, one per token)")
        if not positions.is_cuda or positions.get_device() != self._device:
            raise ValueError(f"Rotary: positions on {positions.device}, frequencies on "
                             f"{self.device}")
        for name, x in (("queries", q), ("keys", k)):
            if x is None:
                continue
            if x.dim() != 3 or x.shape[0] != len(positions) or x.shape[2] != dim:
                raise ValueError(f"Rotary: {name} of shape {tuple(x.shape)}, expected "
                                 f"({len(positions)}, heads, {dim})")
            if x.dtype not in _DTYPE_CODE or x.dtype is not q.dtype:
                raise NotImplementedError(f"Rotary takes bf16, fp16 or fp32 queries and keys of "
                                          f"one type, got {q.dtype} and {x.dtype}")
            _lib.require_current(x, "Rotary")
            if x.get_device() != self._device:
                raise ValueError(f"Rotary: {name} on {x.device}, frequencies on {self.device}")
        q = q if q.stride(2) == 1 else q.contiguous()
        if k is not None:
            k = k if k.stride(2) == 1 else k.contiguous()
        return q, k, positions.contiguous()
