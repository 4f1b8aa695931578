"""Linears that run in 8-bit integers: what an 8-bit per-channel quantization
made (``W_int`` and one scale per output channel) multiplied with tokens
quantized on the fly, one scale (and zero point) per token.

    Y[t, n] = s_t · w_n · (Σ_k c[t, k]·W[n, k] − z_t·Σ_k W[n, k]) + b_n

The integer sums are exact.  Their conversion, the two scales and the bias
round in fp32, then the result to its type.  The token grid is the weight quantizer's (``quant_utils``) at
8 bits with one group per token.  Inference only: nothing here has a
gradient.
"""
import math

import torch

from . import _lib

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32
MAX_COLUMNS = 65536  # longer rows could overflow the 32-bit sums
_MAX_PITCH = (1 << 20) - 16  # bytes between rows of codes


def _rows(x, columns, what):
    """``x`` (..., columns) as a (T, columns) GPU tensor with contiguous rows."""
    if x.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"{what} takes bf16, fp16 or fp32 tokens, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] != columns:
        raise ValueError(f"{what}: tokens of shape {tuple(x.shape)} where the last dimension "
                         f"should be {columns}")
    _lib.require_current(x, what)
    x2 = x if x.dim() == 2 else x.reshape(-1, columns)
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < columns):
        x2 = x2.contiguous()
    return x2


def _row_stride(x2):
    """The row stride of a (T, K) tensor; a single row's is arbitrary in torch."""
    return x2.stride(0) if x2.shape[0] > 1 else max(x2.stride(0), x2.shape[1])


def _padded(n, to=16):
    return (n + to - 1) // to * to


def quantize_tokens(x, sym=True):
    """Codes (int8, shape of ``x``), scale and zero point (fp32, shape of ``x``
    without its last dimension; the zero point is None in the symmetric grid)
    of every token.  A token's value is ``scale · (code − zero)``.

    Codes come as a view of rows padded to 16 bytes, as ``int8_matmul`` reads
    them."""
    columns = x.shape[-1] if x.dim() else 0
    if not 1 <= columns <= MAX_COLUMNS:
        raise ValueError(f"quantize_tokens: rows of 1 to {MAX_COLUMNS} values, got {columns}")
    x2 = _rows(x, columns, "quantize_tokens")
    rows, ldc = x2.shape[0], _padded(columns)
    codes = torch.empty(rows, ldc, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=_F32, device=x.device)
    zero = None if sym else torch.empty(rows, dtype=_F32, device=x.device)
    _lib.call("g2ptq_quantize_tokens", _lib.stream_ptr(x.device), _lib.ptr(x2),
              _DTYPE_CODE[x.dtype], rows, columns, _row_stride(x2), int(bool(sym)),
              _lib.ptr(codes), ldc, _lib.ptr(scale), _lib.ptr(zero))
    lead = x.shape[:-1]
    # (views of the padded rows, also where there is no or more than one leading dimension)
    codes = codes[:, :columns]
    if len(lead) != 1:
        codes = codes.unflatten(0, lead) if lead else codes[0]
    return codes, scale.view(lead), (None if zero is None else zero.view(lead))


class Int8Linear(torch.nn.Module):
    """``y = x̂ · Ŵᵀ + b`` with x̂ the tokens quantized to 8 bits and Ŵ = scale · codes.

    ``codes``: (out, in) int8 GPU tensor; ``scale``: one per output channel;
    ``bias``: (out,) or None; ``sym``: the tokens' grid.  ``y`` has ``x``'s
    dtype.  Columns are laid out once in rows of a multiple of 256 bytes."""

    def __init__(self, codes, scale, bias=None, sym=True):
        super().__init__()
        if codes.dtype is not torch.int8 or codes.dim() != 2:
            raise ValueError(f"Int8Linear takes (out, in) int8 codes, got {codes.dtype} of shape "
                             f"{tuple(codes.shape)}")
        self.out_features, self.in_features = codes.shape
        if not 1 <= self.in_features <= MAX_COLUMNS:
            raise ValueError(f"Int8Linear takes 1 to {MAX_COLUMNS} columns, got "
                             f"{self.in_features}")
        if scale.numel() != self.out_features:
            raise ValueError(f"Int8Linear takes one scale per output channel "
                             f"({self.out_features}), got shape {tuple(scale.shape)}")
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError(f"Int8Linear: bias of shape {tuple(bias.shape)}, expected "
                             f"({self.out_features},)")
        if not codes.is_cuda:
            raise RuntimeError("Int8Linear requires GPU tensors")
        self.sym = bool(sym)
        dev = codes.device
        self._shape = (self.out_features, _padded(self.in_features, 256))
        weight = torch.zeros(self._shape, dtype=torch.int8, device=dev)
        weight[:, :self.in_features] = codes
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", scale.detach().reshape(-1).to(
            device=dev, dtype=torch.float32, copy=True))
        self.register_buffer("weight_sum", None if self.sym else
                             codes.sum(dim=1, dtype=torch.int32))
        self.register_buffer("bias", None if bias is None else bias.detach().to(
            device=dev, dtype=torch.float32, copy=True))

    def _apply(self, fn, recurse=True):
        """The module follows its model to another device; a cast of the model leaves it as it
        is: the kernels read int8 codes and fp32 scales and biases, whatever the tokens' type."""
        before = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, was in before.items():
            now = self._buffers[name]
            if now is not None and now.dtype is not was.dtype:
                self._buffers[name] = was.to(now.device)
        return self

    def _operands(self):
        """The weights, scales, sums and biases (the last two or None) and their device's index.
        The kernels know them by their addresses, and buffers can be replaced by any tensor
        (``load_state_dict`` with ``assign``, an attribute set), so every call looks at them."""
        held, n, shape = self._buffers, self.out_features, self._shape
        # (attribute access of a module's buffers is slow)
        weight, scale, total, bias = (held["weight"], held["weight_scale"], held["weight_sum"],
                                      held["bias"])
        here = weight.get_device()
        if not (weight.dtype is _I8 and weight.shape == shape and weight.is_contiguous()
                and scale.dtype is _F32 and scale.numel() == n and scale.is_contiguous()
                and scale.get_device() == here
                and (bias is None or (bias.dtype is _F32 and bias.numel() == n
                                      and bias.is_contiguous() and bias.get_device() == here))
                and (total is None or (total.dtype is _I32 and total.numel() == n
                                       and total.is_contiguous()
                                       and total.get_device() == here))):
            for name, dtype, size in (("weight", _I8, shape), ("weight_scale", _F32, (n,)),
                                      ("weight_sum", _I32, (n,)), ("bias", _F32, (n,))):
                t = held[name]
                if t is not None and (t.dtype is not dtype or t.numel() != math.prod(size)
                                      or (name == "weight" and t.shape != shape)
                                      or not t.is_contiguous() or t.get_device() != here):
                    raise ValueError(f"Int8Linear: {name} is {t.dtype} of shape {tuple(t.shape)} "
                                     f"and strides {t.stride()} on {t.device}; a contiguous "
                                     f"{dtype} tensor of shape {size} on {weight.device} is "
                                     "needed")
        return weight, scale, total, bias, here

    @classmethod
    def from_export(cls, qparams, bias=None, sym=True, bits=None):
        """From a layer's exported tensors (``layer._export_qparams`` of a symmetric 8-bit
        ``fasterquant(..., export_compressed_tensors=True)`` with one group per row, or the
        buffers that ``register_qparam_buffers`` made of them): the layer itself, or a dict
        of them.

        The tensors do not tell the codes' width.  A layer that was exported here knows it;
        where nothing does, codes without a single bit that narrower ones cannot have are
        refused unless ``bits=8`` vouches for them."""
        grid = None
        if isinstance(qparams, torch.nn.Module):
            layer = qparams
            grid = layer.__dict__.get("_export_grid")
            qparams = layer.__dict__.get("_export_qparams") or {
                k: b for k, b in layer.named_buffers(recurse=False)}
            bias = getattr(layer, "bias", None) if bias is None else bias
        if bits not in (None, 8) or (grid and grid[0] != 8):
            raise ValueError(f"Int8Linear.from_export: codes of "
                             f"{bits if bits not in (None, 8) else grid[0]} bits are no 8-bit codes")
        if grid and grid[1] is False:
            raise ValueError("Int8Linear.from_export: an asymmetric quantization's export holds "
                             "codes without their zero points; quantize with sym=True")
        try:
            packed, scale = qparams["weight_packed"], qparams["weight_scale"]
            rows, columns = (int(n) for n in qparams["weight_shape"])
        except KeyError as e:
            raise ValueError(f"Int8Linear.from_export: no {e} among the exported tensors") from None
        if packed.shape != (rows, (columns + 3) // 4):
            raise ValueError(f"Int8Linear.from_export: packed words of shape "
                             f"{tuple(packed.shape)} are no 8-bit codes of a {rows}x{columns} "
                             "weight")
        if scale.numel() != rows:
            raise ValueError(f"Int8Linear.from_export: scales of shape {tuple(scale.shape)}; "
                             "one group per row (groupsize -1) is needed")
        # 7-bit codes lie four to a word as well, narrower ones too in rows of up to four: none
        # reaches past bit 7n of a word of n codes
        if bits is None and grid is None and packed.numel():
            n = min(columns, 4)
            if not bool(((packed >> (7 * n)) & ((1 << n) - 1)).any()):
                raise ValueError("Int8Linear.from_export: the packed words look like codes of 7 "
                                 "bits or fewer, not like 8-bit codes; bits=8 if they are")
        codes = packed.contiguous().view(torch.uint8)[:, :columns]
        return cls((codes ^ 0x80).view(torch.int8), scale, bias=bias, sym=sym)

    @classmethod
    def from_linear(cls, linear, quantizer, sym=True):
        """Round-to-nearest codes of ``linear.weight`` on a fitted symmetric
        per-channel ``WeightQuantizer`` of at most 8 bits."""
        if not quantizer.ready() or quantizer.bits > 8 or not quantizer.sym \
                or quantizer.weight_groupsize > 0:
            raise ValueError("Int8Linear.from_linear needs a fitted symmetric per-channel "
                             "quantizer of at most 8 bits")
        weight = linear.weight.detach()
        _, codes, scale = quantizer.fake_quantize(weight)
        if scale.numel() == 1:
            scale = scale.reshape(1).expand(weight.shape[0])
        return cls(codes.to(torch.int8), scale, bias=linear.bias, sym=sym)

    def forward(self, x):
        columns, out = self.in_features, self.out_features
        weight, scale, total, bias, here = self._operands()
        # what is usual passes in one go (a call is a few microseconds); the rest is told apart
        if (x.dim() == 2 and x.shape[1] == columns and x.is_contiguous()
                and x.dtype in _DTYPE_CODE and not x.requires_grad
                and _lib.forward_ad._current_level < 0
                and x.get_device() == here == torch._C._cuda_getDevice()):
            x2, rows, stride = x, x.shape[0], columns
        else:
            x2 = _rows(x, columns, "Int8Linear")
            if here != x.get_device():
                raise ValueError(f"Int8Linear: tokens on {x.device}, weights on {weight.device}")
            rows, stride = x2.shape[0], _row_stride(x2)
        y = x.new_empty((rows, out))
        if rows:
            need = _lib.workspace_fast("int8_linear_workspace", rows, out, columns)
            ws = _lib.scratch(need, x.device) if need else None
            _lib.call_fast("int8_linear", _lib.current_stream(), x2.data_ptr(),
                           _DTYPE_CODE[x.dtype], rows, columns, stride, self.sym,
                           weight.data_ptr(), self._shape[1], scale.data_ptr(),
                           None if total is None else total.data_ptr(),
                           None if bias is None else bias.data_ptr(), out, y.data_ptr(), out,
                           None if ws is None else ws.data_ptr(), need)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], out)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, sym={self.sym}")


def int8_matmul(codes, scale, linear, zero=None, dtype=torch.bfloat16):
    """The product alone, for tokens that several linears share: ``codes``,
    ``scale`` and ``zero`` from ``quantize_tokens``, ``linear`` an
    ``Int8Linear``; the result is what ``linear`` gives for the tokens, in
    ``dtype``."""
    if codes.dtype is not torch.int8 or codes.dim() == 0 \
            or codes.shape[-1] != linear.in_features:
        raise ValueError(f"int8_matmul: codes of {codes.dtype} and shape {tuple(codes.shape)} for "
                         f"{linear.in_features} columns")
    if dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"int8_matmul gives bf16, fp16 or fp32, not {dtype}")
    _lib.require_current(codes, "int8_matmul")
    lead, columns, out = codes.shape[:-1], linear.in_features, linear.out_features
    for name, t in (("scale", scale), ("zero", zero)):
        if t is not None and (t.dtype is not torch.float32 or t.shape != lead):
            raise ValueError(f"int8_matmul: {name} of {t.dtype} and shape {tuple(t.shape)}, "
                             f"expected fp32 {tuple(lead)}")
        if t is not None and t.get_device() != codes.get_device():
            raise ValueError(f"int8_matmul: {name} on {t.device}, codes on {codes.device}")
    weight, wscale, total, bias, here = linear._operands()
    if here != codes.get_device():
        raise ValueError(f"int8_matmul: codes on {codes.device}, weights on {weight.device}")
    if zero is not None and total is None:
        raise ValueError("int8_matmul: tokens with zero points need a linear made with sym=False")
    c2 = codes if codes.dim() == 2 else codes.flatten(0, -2) if codes.dim() > 2 \
        else codes.unsqueeze(0)
    rows, need = c2.shape[0], _padded(columns)
    # rows have to be readable in 16-byte steps to their end, and at most _MAX_PITCH apart (a
    # tile's offsets are 32-bit); others are laid out again
    room = c2.untyped_storage().nbytes() - c2.storage_offset()
    if (c2.stride(1) != 1 or c2.stride(0) % 16 or not need <= c2.stride(0) <= _MAX_PITCH
            or c2.data_ptr() % 16 or (rows - 1) * c2.stride(0) + need > room):
        padded = torch.zeros(rows, need, dtype=torch.int8, device=codes.device)
        padded[:, :columns] = c2
        c2 = padded
    y = torch.empty(rows, out, dtype=dtype, device=codes.device)
    if rows:
        scale, zero = scale.contiguous(), None if zero is None else zero.contiguous()
        _lib.call("g2ptq_int8_gemm", _lib.stream_ptr(codes.device), _lib.ptr(c2), c2.stride(0),
                  _lib.ptr(scale), _lib.ptr(zero), _lib.ptr(weight), linear._shape[1],
                  _lib.ptr(wscale), _lib.ptr(None if zero is None else total), _lib.ptr(bias),
                  rows, out, columns, _lib.ptr(y), _DTYPE_CODE[dtype], out, None, 0)
    return y.view(*lead, out)
