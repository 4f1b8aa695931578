"""Root-mean-square norm of tokens, with the residual's addition, and its 8-bit codes.

    s = x + residual,  y_c = s_c · w_c / sqrt(mean(s²) + eps)

One pass over the data; sums, the root and ``y`` are fp32, and ``s`` and ``y`` are rounded once
where they are returned.  ``rms_norm_quantize`` gives ``y`` (before that rounding) on the token
grid of ``quantize_tokens``, as ``int8_matmul`` takes it for the projections that share it.
Inference only: nothing here has a gradient.
"""
from collections import namedtuple

import torch

from . import _lib
from .int8_utils import _DTYPE_CODE, MAX_COLUMNS, _padded

_F32, _CONTIGUOUS = torch.float32, torch.contiguous_format
NormedTokens = namedtuple("NormedTokens", "codes scale zero values sum")


def _rows(x, what):
    """``x`` (copied where two strides do not tell its rows), their number, how many of them
    lie one inner stride apart, and the outer and the inner stride."""
    columns = x.shape[-1]
    if x.is_contiguous():
        return x, x.numel() // columns, 1, columns, 0
    if x.stride(-1) == 1 or columns == 1:
        dims = []  # of rows, the innermost first; dimensions that continue each other are one
        for size, stride in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
            if size == 1:
                continue
            if dims and stride == dims[-1][0] * dims[-1][1]:
                dims[-1] = (dims[-1][0] * size, dims[-1][1])
            else:
                dims.append((size, stride))
        if len(dims) == 1:
            return x, dims[0][0], 1, dims[0][1], 0
        if len(dims) == 2:
            (inner, si), (outer, so) = dims
            return x, inner * outer, inner, so, si
    x = x.contiguous()
    return x, x.numel() // columns, 1, columns, 0


def _check(x, weight, eps, residual, what):
    if x.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"{what} takes bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_COLUMNS:
        raise ValueError(f"{what}: rows of 1 to {MAX_COLUMNS} values, got shape {tuple(x.shape)}")
    _lib.require_current(x, what)
    if weight.dtype not in _DTYPE_CODE or tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"{what}: a weight of {weight.dtype} and shape {tuple(weight.shape)} for "
                         f"{x.shape[-1]} columns (bf16, fp16 or fp32, one per column)")
    _lib.require_current(weight, what)
    if not 0 <= eps < float("inf"):
        raise ValueError(f"{what}: eps is {eps}")
    if residual is not None:
        if residual.dtype is not x.dtype or residual.shape != x.shape:
            raise ValueError(f"{what}: a residual of {residual.dtype} and shape "
                             f"{tuple(residual.shape)} for {x.dtype} of shape {tuple(x.shape)}")
        _lib.require_current(residual, what)


def _norm(x, weight, eps, residual, y, total, sym, codes, ldc, scale, zero, what):
    x, rows, inner, xo, xi = _rows(x, what)
    r = ro = ri = None
    if residual is not None:
        residual, _, r_inner, ro, ri = _rows(residual, what)
        if r_inner != inner:
            # rows of one of the two follow each other without a gap: give both the same pairs
            if inner == 1:
                inner, xo, xi = r_inner, xo * r_inner, xo
            elif r_inner == 1:
                ro, ri = ro * inner, ro
            else:
                residual = residual.contiguous()
                ri = x.shape[-1]
                ro = ri * inner
        r = residual.data_ptr()
    if rows:
        weight = weight if weight.is_contiguous() else weight.contiguous()
        _lib.call_fast("rms_norm", _lib.current_stream(), x.data_ptr(), xo, xi, r, ro or 0,
                       ri or 0, _DTYPE_CODE[x.dtype], weight.data_ptr(),
                       _DTYPE_CODE[weight.dtype], rows, inner, x.shape[-1], eps,
                       None if y is None else y.data_ptr(),
                       None if total is None else total.data_ptr(), sym,
                       None if codes is None else codes.data_ptr(), ldc,
                       None if scale is None else scale.data_ptr(),
                       None if zero is None else zero.data_ptr())


def _usual(x, weight, residual):
    """Whether the arguments pass all checks in one go and lie as the kernel takes them (a call
    is a few microseconds); what is not is looked at one by one."""
    here, dtype = x.get_device(), x.dtype
    return (x.numel() and x.dim() and weight.dim() == 1 and weight.shape[0] == x.shape[-1]
            and dtype in _DTYPE_CODE and weight.dtype in _DTYPE_CODE
            and x.is_contiguous() and weight.is_contiguous()
            and here == weight.get_device() == torch._C._cuda_getDevice()
            and _lib.forward_ad._current_level < 0
            and (residual is None or (residual.dtype is dtype and residual.shape == x.shape
                                      and residual.is_contiguous()
                                      and residual.get_device() == here
                                      and not (residual.requires_grad
                                               and torch.is_grad_enabled())))
            and not ((x.requires_grad or weight.requires_grad) and torch.is_grad_enabled()))


def rms_norm(x, weight, eps=1e-6, residual=None):
    """``y`` of every row of ``x`` (..., C; bf16, fp16 or fp32), in its type; with a
    ``residual`` (``x``'s shape and type) the pair ``(y, s)``.

    ``weight`` (C,) is bf16, fp16 or fp32.  Rows may be strided (a projection's heads).  ``y``
    is the norm of the sum before ``s`` is rounded.  A row of zeros is NaN with ``eps=0``; a
    NaN makes its row NaN."""
    if x.is_cuda and _usual(x, weight, residual):
        columns, code = x.shape[-1], _DTYPE_CODE[x.dtype]
        y = torch.empty_like(x)
        total = None if residual is None else torch.empty_like(x)
        _lib.call_fast("rms_norm", _lib.current_stream(), x.data_ptr(), columns, 0,
                       None if residual is None else residual.data_ptr(), columns, 0, code,
                       weight.data_ptr(), _DTYPE_CODE[weight.dtype], x.numel() // columns, 1,
                       columns, eps, y.data_ptr(), None if total is None else total.data_ptr(),
                       True, None, 0, None, None)
        return y if total is None else (y, total)
    _check(x, weight, eps, residual, "rms_norm")
    y = torch.empty_like(x, memory_format=_CONTIGUOUS)
    total = None if residual is None else torch.empty_like(x, memory_format=_CONTIGUOUS)
    _norm(x, weight, eps, residual, y, total, True, None, 0, None, None, "rms_norm")
    return y if residual is None else (y, total)


def rms_norm_quantize(x, weight, eps=1e-6, residual=None, sym=True, values=False):
    """``rms_norm`` on the 8-bit token grid: ``(codes, scale, zero, values, sum)``.

    ``codes``, ``scale`` and ``zero`` are what ``quantize_tokens`` would make of ``y`` before it
    is rounded to ``x``'s type (``zero`` is None with ``sym``); ``values`` is ``y`` in that type
    if it is asked for, ``sum`` is ``x + residual`` where there is one, else None."""
    usual = x.is_cuda and _usual(x, weight, residual)
    if not usual:
        _check(x, weight, eps, residual, "rms_norm_quantize")
    lead, columns, dev = x.shape[:-1], x.shape[-1], x.device
    rows, ldc = x.numel() // columns, _padded(columns)
    codes = torch.empty(rows, ldc, dtype=torch.int8, device=dev)
    scale = torch.empty(rows, dtype=_F32, device=dev)
    zero = None if sym else torch.empty(rows, dtype=_F32, device=dev)
    y = torch.empty_like(x, memory_format=_CONTIGUOUS) if values else None
    total = None if residual is None else torch.empty_like(x, memory_format=_CONTIGUOUS)
    if usual:
        _lib.call_fast("rms_norm", _lib.current_stream(), x.data_ptr(), columns, 0,
                       None if residual is None else residual.data_ptr(), columns, 0,
                       _DTYPE_CODE[x.dtype], weight.data_ptr(), _DTYPE_CODE[weight.dtype], rows, 1,
                       columns, eps, None if y is None else y.data_ptr(),
                       None if total is None else total.data_ptr(), bool(sym), codes.data_ptr(),
                       ldc, scale.data_ptr(), None if zero is None else zero.data_ptr())
    else:
        _norm(x, weight, eps, residual, y, total, bool(sym), codes, ldc, scale, zero,
              "rms_norm_quantize")
    # (views of the padded rows, as quantize_tokens gives them)
    if ldc != columns:
        codes = codes[:, :columns]
    if len(lead) != 1:
        codes = codes.unflatten(0, lead) if lead else codes[0]
        scale, zero = scale.view(lead), None if zero is None else zero.view(lead)
    return NormedTokens(codes, scale, zero, y, total)
