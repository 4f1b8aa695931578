"""Low-rank adapters of many requests beside a shared projection.

    out_t = base_t + scale_a · up_a · (down_a · x_t),  a = index_t

Every token of a batch may have another adapter, or none.  ``base`` is what the shared
projection (an ``Int8Linear``, say) gives:

    adapters = LowRankAdapters(down, up, scale=alpha / rank)
    y = adapters(x, index, base=proj(x))            # or adapters.add_(y, x, index)

Sums are fp32, the result is rounded once.  Inference only: nothing here has a gradient.
"""
import ctypes

import torch

from . import _lib
from .int8_utils import _padded, _row_stride

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1}
_I32 = torch.int32
MAX_RANK, MAX_FEATURES = 512, 1 << 20


class LowRankAdapters:
    """``down``: n tensors (rank_i, in_features), ``up``: n tensors (out_features, rank_i), all
    bf16 or all fp16 on one GPU, ranks of 1 to 512; ``scale``: a number, or one per adapter.
    They are copied once into the layout of the kernels, which gives every adapter the set's
    largest rank: memory is n times that rank, 16 at least.  A set does not change: other adapters
    are another set, and a graph that was captured with the old one needs it kept.

    Equal calls give equal bits.  The order in which a token's products are summed in fp32 goes by
    the call's number of tokens, not by which tokens they are."""

    def __init__(self, down, up, scale=1.0):
        down, up = list(down), list(up)
        n = len(down)
        if n == 0 or len(up) != n:
            raise ValueError(f"LowRankAdapters: {n} down and {len(up)} up matrices")
        first = down[0]
        if first.dtype not in _DTYPE_CODE:
            raise NotImplementedError(f"LowRankAdapters holds bf16 or fp16, not {first.dtype}")
        if not first.is_cuda:
            raise RuntimeError("LowRankAdapters live on the GPU")
        if first.dim() != 2 or up[0].dim() != 2:
            raise ValueError("LowRankAdapters takes matrices")
        self.in_features, self.out_features = first.shape[1], up[0].shape[0]
        if not (1 <= self.in_features <= MAX_FEATURES and 1 <= self.out_features <= MAX_FEATURES):
            raise ValueError(f"LowRankAdapters: {self.in_features} to {self.out_features} features "
                             f"(1 to {MAX_FEATURES})")
        for i, (d, u) in enumerate(zip(down, up)):
            if d.dtype is not first.dtype or u.dtype is not first.dtype \
                    or d.device != first.device or u.device != first.device:
                raise ValueError(f"LowRankAdapters: adapter {i} is {d.dtype} on {d.device} and "
                                 f"{u.dtype} on {u.device}, the first {first.dtype} on "
                                 f"{first.device}")
            if d.dim() != 2 or u.dim() != 2 or d.shape[1] != self.in_features \
                    or u.shape != (self.out_features, d.shape[0]) \
                    or not 1 <= d.shape[0] <= MAX_RANK:
                raise ValueError(f"LowRankAdapters: adapter {i} of shapes {tuple(d.shape)} and "
                                 f"{tuple(u.shape)} for {self.in_features} to "
                                 f"{self.out_features} features (ranks of 1 to {MAX_RANK})")
        scales = torch.as_tensor(scale, dtype=torch.float64).detach().flatten().cpu()
        if scales.numel() not in (1, n):
            raise ValueError(f"LowRankAdapters: {scales.numel()} scales for {n} adapters")
        self.ranks = tuple(d.shape[0] for d in down)
        self.dtype, self.device = first.dtype, first.device
        self._device = self.device.index
        R, dev = _padded(max(self.ranks)), self.device
        with torch.no_grad():
            d = torch.zeros(n, R, _padded(self.in_features, 64), dtype=self.dtype, device=dev)
            u = torch.zeros(n, _padded(self.out_features, 64), R, dtype=self.dtype, device=dev)
            for i, r in enumerate(self.ranks):
                d[i, :r, :self.in_features] = down[i]
                u[i, :self.out_features, :r] = up[i]
            # (a rare set: kernels of its own look after these weights)
            infinite = bool(u.isinf().any())
            # the order in which the kernels' lanes take 16 bytes each: down by 16 ranks and 64
            # columns (2 × 4 × 16 pieces: half of 16 columns, 16 columns, rank), up by 64 channels
            # and 16 ranks (4 × 2 × 16: 16 channels, half of the ranks, channel)
            d = d.view(n, R // 16, 16, -1, 4, 2, 8).permute(0, 1, 3, 5, 4, 2, 6).contiguous()
            u = u.view(n, -1, 4, 16, R // 16, 2, 8).permute(0, 1, 4, 2, 5, 3, 6).contiguous()
        self._held = (d, u, torch.tensor(self.ranks, dtype=_I32, device=dev),
                      scales.expand(n).to(torch.float32).contiguous().to(dev),
                      torch.zeros(1, dtype=_I32, device=dev))
        self._struct = _lib.AdapterSetStruct(*(_lib.ptr(t) for t in self._held), n, R,
                                             self.in_features, self.out_features,
                                             _DTYPE_CODE[self.dtype]
                                             | (_lib.ADAPTERS_INFINITE if infinite else 0))
        self._address = ctypes.addressof(self._struct)
        self._n, self._rank = n, R

    def __len__(self):
        return self._n

    flags = property(lambda self: self._held[4])

    def _rows(self, t, columns, what):
        """``t`` as a (tokens, columns) tensor of contiguous rows."""
        if t.dtype is not self.dtype:
            raise NotImplementedError(f"LowRankAdapters of {self.dtype} takes {what} of that type, "
                                      f"got {t.dtype}")
        if t.dim() == 0 or t.shape[-1] != columns:
            raise ValueError(f"LowRankAdapters: {what} of shape {tuple(t.shape)} where the last "
                             f"dimension should be {columns}")
        _lib.require_current(t, "LowRankAdapters")
        if t.get_device() != self._device:
            raise ValueError(f"LowRankAdapters: {what} on {t.device}, the adapters on "
                             f"{self.device}")
        return t if t.dim() == 2 else t.reshape(-1, columns)

    def _run(self, x, index, base, out):
        """``base`` and ``out`` with contiguous rows, (tokens, out_features)."""
        rows = x.shape[0]
        if x.stride(1) != 1 and x.shape[1] != 1:
            x = x.contiguous()
        index = index.reshape(-1)
        index = index if index.is_contiguous() else index.contiguous()
        if rows:
            need = _lib.workspace_fast("adapters_workspace", rows, self.in_features, self._n,
                                       self._rank)
            ws = _lib.scratch(need, self.device)
            _lib.call_fast("adapters", _lib.current_stream(), self._address, x.data_ptr(),
                           x.stride(0), index.data_ptr(), rows,
                           None if base is None else base.data_ptr(),
                           0 if base is None else base.stride(0), out.data_ptr(), out.stride(0),
                           ws.data_ptr(), need)

    def _index(self, index, lead):
        if index.dtype is not _I32 or index.shape != lead:
            raise ValueError(f"LowRankAdapters: an index of {index.dtype} and shape "
                             f"{tuple(index.shape)}, expected int32 of shape {tuple(lead)}")
        if index.get_device() != self._device:
            raise ValueError(f"LowRankAdapters: the index on {index.device}, the adapters on "
                             f"{self.device}")

    def __call__(self, x, index, base=None):
        """``base`` (..., out_features; None: zeros) plus each token's own adapter's part, as a
        new tensor.  ``x`` (..., in_features) and ``base`` have the adapters' type; ``index``
        (int32, ``x``'s shape without its last dimension) is each token's adapter, negative
        for none.  An index of no adapter counts as none and is flagged."""
        dtype, here, rows, out = self.dtype, self._device, index.numel(), self.out_features
        # what is usual passes in one go (a call is a few microseconds); the rest is told apart
        if (rows and base is not None and x.dim() == 2 and x.dtype is base.dtype is dtype
                and index.dtype is _I32 and x.shape == (rows, self.in_features)
                and base.shape == (rows, out) and index.dim() == 1 and x.is_contiguous()
                and base.is_contiguous() and index.is_contiguous()
                and x.get_device() == base.get_device() == index.get_device() == here
                and torch._C._cuda_getDevice() == here
                and not x.requires_grad and not base.requires_grad
                and _lib.forward_ad._current_level < 0):
            y = torch.empty_like(base)
            need = _lib.workspace_fast("adapters_workspace", rows, self.in_features, self._n,
                                       self._rank)
            ws = _lib.scratch(need, self.device)  # (held until the launch)
            _lib.call_fast("adapters", _lib.current_stream(), self._address, x.data_ptr(),
                           self.in_features, index.data_ptr(), rows, base.data_ptr(), out,
                           y.data_ptr(), out, ws.data_ptr(), need)
            return y
        lead = x.shape[:-1]
        x2 = self._rows(x, self.in_features, "tokens")
        self._index(index, lead)
        b2 = None
        if base is not None:
            b2 = self._rows(base, out, "a base")
            if base.shape[:-1] != lead:
                raise ValueError(f"LowRankAdapters: a base of shape {tuple(base.shape)} for tokens "
                                 f"of shape {tuple(x.shape)}")
            if b2.stride(1) != 1 and out != 1:
                b2 = b2.contiguous()
        y = torch.empty(x2.shape[0], out, dtype=self.dtype, device=self.device)
        self._run(x2, index, b2, y)
        return y if x.dim() == 2 else y.view(*lead, out)

    def add_(self, y, x, index):
        """The same in place: each token's own adapter's part is added to its row of ``y``
        (..., out_features), whose rows may be strided; rows without an adapter are not touched.
        Returns ``y``."""
        lead = x.shape[:-1]
        x2 = self._rows(x, self.in_features, "tokens")
        self._index(index, lead)
        if y.shape[:-1] != lead:
            raise ValueError(f"LowRankAdapters.add_: an output of shape {tuple(y.shape)} for tokens "
                             f"of shape {tuple(x.shape)}")
        y2 = self._rows(y, self.out_features, "an output")
        rows = y2.shape[0]
        if rows and (y2.data_ptr() != y.data_ptr()
                     or (y2.stride(1) != 1 and y2.shape[1] != 1)
                     or (rows > 1 and y2.stride(0) < y2.shape[1])):
            raise ValueError(f"LowRankAdapters.add_: an output of strides {y.stride()} (contiguous "
                             "rows, one stride apart that do not overlap, are needed)")
        self._run(x2, index, y2, y2)
        return y

    def check(self):
        """Raise if an index of no adapter was met since the last check (waits for the current
        stream)."""
        v = int(self.flags.item())
        self.flags.zero_()
        if v & _lib.FLAG_BAD_INDEX:
            raise IndexError(f"an index outside {self._n} adapters was given to LowRankAdapters")
