"""A paged cache of quantized keys and values, and attention over it.

Keys and values are quantized as they are written, with 4 or 8 bits on the
weight quantizer's grid (``quant_utils``), one scale (and zero point) per token
and head.  A slot is ``page number · page_size + offset``; a sequence's token p
lives in slot ``table[b, p // page_size] · page_size + p % page_size``.

    cache = PagedKVCache(num_pages, page_size=64, kv_heads=8, head_dim=128, bits=4, sym=False)
    cache.write(k, v, slots)                       # this step's tokens
    out = paged_attention(q, cache, table, cu_q, kv_lens)
    k, v = cache.read(table, cu_tokens, total)     # what the cache stands for

Page tables, offsets and lengths are device tensors: nothing here waits for
the GPU, and a step can be captured into a graph.  Indices outside the cache
are never followed; they are flagged, and ``cache.check()`` raises for them at
a point of the caller's choosing.  Inference only: nothing has a gradient.
"""
import ctypes
import math

import torch

from . import _lib

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _heads(x, heads, dim, what):
    """``x`` (tokens, heads, dim) with contiguous channels on the GPU."""
    shape = x.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{what} of shape {tuple(shape)}, expected (tokens, {heads}, {dim})")
    _lib.require_current(x, what)
    return x if x.stride(2) == 1 else x.contiguous()


def _index(t, dtype, dims, what, device):
    if t.dtype is not dtype or t.dim() != dims:
        raise ValueError(f"{what}: a {dims}-dimensional {dtype} tensor is needed, got "
                         f"{t.dtype} of shape {tuple(t.shape)}")
    if not t.is_cuda or t.get_device() != device.index:
        raise ValueError(f"{what} on {t.device}, the cache on {device}")
    return t if t.is_contiguous() or _rows_apart(t) else t.contiguous()


def _rows_apart(t):
    return t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` slots for ``kv_heads`` heads of
    ``head_dim`` channels, keys and values, ``bits`` 4 or 8.

    ``k_codes``, ``v_codes`` (num_pages, kv_heads, page_size, head_dim·bits/8)
    uint8, ``k_scale``, ``v_scale`` (num_pages, kv_heads, page_size) fp32 and,
    with ``sym=False``, ``k_zero``, ``v_zero`` uint8 hold the cache; a code u
    stands for ``scale · (u − zero)`` with ``zero = 2^(bits − 1)`` in the
    symmetric grid.  Slots never written stand for zeros."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, bits=8, sym=True, device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"PagedKVCache holds 4 or 8 bits, not {bits}")
        if page_size < 1 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: pages of {page_size} slots (a power of two up to "
                             "4096 is needed)")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"PagedKVCache: head dimension {head_dim} (a multiple of 16 up to "
                             "256 is needed)")
        if num_pages < 0 or not 1 <= kv_heads <= 65535:
            raise ValueError(f"PagedKVCache: {num_pages} pages of {kv_heads} heads")
        if num_pages * kv_heads * page_size >= 1 << 31:
            raise ValueError(f"PagedKVCache: {num_pages} pages of {kv_heads} heads of {page_size} "
                             "slots (fewer than 2^31 in all)")
        self.num_pages, self.page_size = num_pages, page_size
        self.kv_heads, self.head_dim, self.bits, self.sym = kv_heads, head_dim, bits, bool(sym)
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("PagedKVCache lives on the GPU")
        shape = (num_pages, kv_heads, page_size)
        codes = [torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=dev)
                 for _ in range(2)]
        scales = [torch.zeros(shape, dtype=torch.float32, device=dev) for _ in range(2)]
        zeros = [None if self.sym else torch.zeros(shape, dtype=torch.uint8, device=dev)
                 for _ in range(2)]
        flags = torch.zeros(1, dtype=torch.int32, device=dev)
        self.device = flags.device
        self._device = self.device.index
        self._held = (*codes, *scales, *zeros, flags)
        self._struct = _lib.KvCacheStruct(
            *(_lib.ptr(t) for t in self._held),
            num_pages, kv_heads, page_size, head_dim, bits, int(self.sym))
        self._address = ctypes.addressof(self._struct)

    # (the kernels know these by their addresses: changed in place, never replaced)
    k_codes, v_codes, k_scale, v_scale, k_zero, v_zero, flags = (
        property(lambda self, i=i: self._held[i]) for i in range(7))

    def write(self, k, v, slots):
        """Quantize tokens' keys and values (tokens, kv_heads, head_dim; bf16, fp16
        or fp32, any strides of token and head) into their slots (int64).
        Negative slots are skipped (padding of a batch); slots must not repeat
        within a call."""
        here, code = self._device, _DTYPE_CODE.get(k.dtype)
        # what is usual passes in one go (a call is a few microseconds); the rest is told apart
        if not (slots.dim() == 1 and slots.dtype is torch.int64 and slots.is_contiguous()
                and k.shape == v.shape == (slots.shape[0], self.kv_heads, self.head_dim)
                and k.stride(2) == v.stride(2) == 1 and code is not None and v.dtype is k.dtype
                and k.get_device() == v.get_device() == slots.get_device() == here
                and torch._C._cuda_getDevice() == here
                and not k.requires_grad and not v.requires_grad
                and _lib.forward_ad._current_level < 0):
            return self._write_checked(k, v, slots)
        (n, _, _), (kt, kh, _), (vt, vh, _) = k.shape, k.stride(), v.stride()
        _lib.call_fast("kv_write", _lib.current_stream(), self._address, k.data_ptr(), kt, kh,
                       v.data_ptr(), vt, vh, code, n, slots.data_ptr())

    def _write_checked(self, k, v, slots):
        k = _heads(k, self.kv_heads, self.head_dim, "keys")
        v = _heads(v, self.kv_heads, self.head_dim, "values")
        if k.dtype not in _DTYPE_CODE or v.dtype is not k.dtype:
            raise NotImplementedError(f"PagedKVCache.write takes bf16, fp16 or fp32 keys and "
                                      f"values, got {k.dtype} and {v.dtype}")
        slots = _index(slots, torch.int64, 1, "slots", self.device)
        n = len(k)
        if n != len(v) or n != len(slots):
            raise ValueError(f"{n} keys, {len(v)} values, {len(slots)} slots")
        if k.get_device() != self._device:
            raise ValueError(f"keys on {k.device}, the cache on {self.device}")
        (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
        _lib.call_fast("kv_write", _lib.current_stream(), self._address, k.data_ptr(), kt, kh,
                       v.data_ptr(), vt, vh, _DTYPE_CODE[k.dtype], n, slots.data_ptr())

    def read(self, table, cu_tokens, total, dtype=torch.bfloat16):
        """``(k, v)``, each (total, kv_heads, head_dim) of ``dtype``: rows
        ``cu_tokens[b]`` to ``cu_tokens[b + 1]`` hold the first positions of the
        sequence whose pages are ``table[b]`` (both int32).  Rows outside every
        sequence, and positions without a page, are zero."""
        here, cu = self._device, cu_tokens
        # (as in write)
        if not (table.dtype is cu.dtype is torch.int32 and table.dim() == 2 and cu.dim() == 1
                and table.is_contiguous() and cu.is_contiguous()
                and table.get_device() == cu.get_device() == here
                and torch._C._cuda_getDevice() == here):
            table = _index(table, torch.int32, 2, "table", self.device)
            cu = _index(cu, torch.int32, 1, "cu_tokens", self.device)
            _lib.require_current(self._held[6], "PagedKVCache.read")
        if dtype not in _DTYPE_CODE:
            raise NotImplementedError(f"PagedKVCache.read gives bf16, fp16 or fp32, not {dtype}")
        B, width = table.shape
        if cu.shape[0] != B + 1:
            raise ValueError(f"cu_tokens has {cu.shape[0]} entries for {B} sequences")
        if total < 0:
            raise ValueError(f"total is {total}")
        k = torch.empty(total, self.kv_heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _lib.call_fast("kv_read", _lib.current_stream(), self._address, table.data_ptr(),
                       max(table.stride(0), width), B, width, cu.data_ptr(), total, k.data_ptr(),
                       v.data_ptr(), _DTYPE_CODE[dtype])
        return k, v

    def check(self):
        """Raise if a slot or page outside the cache was met since the last check, by the
        work that the current stream has or waits for (waits for that stream)."""
        v = int(self.flags.item())
        self.flags.zero_()
        if v & _lib.FLAG_BAD_INDEX:
            raise IndexError("a slot or page outside the cache was given to a PagedKVCache")


def paged_attention(q, cache, table, cu_q, kv_lens, scale=None, max_q=None, max_kv=None):
    """Causal attention of each sequence's new tokens over its keys and values in
    the cache (the new tokens' own among them: write before attending).

    ``q`` (tokens, heads, head_dim) bf16 or fp16, any strides of token and
    head: rows ``cu_q[b]`` to ``cu_q[b + 1]`` are the last tokens of sequence b,
    which has ``kv_lens[b]`` in the cache, in pages ``table[b]`` (all int32).
    ``heads`` is a multiple of the cache's; neighbouring heads share one of them.
    ``scale`` defaults to 1/sqrt(head_dim).  Returns (tokens, heads, head_dim) in
    ``q``'s dtype; rows without a key, and rows outside every sequence, are zero.

    ``max_q`` and ``max_kv``, the batch's most new tokens and longest sequence
    where the caller knows them, size the launch (default: all tokens, the whole
    table); lengths beyond them are still computed."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"paged_attention takes bf16 or fp16 queries, got {q.dtype}")
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"queries of shape {tuple(q.shape)} over {cache.kv_heads} heads of the "
                         "cache")
    q = _heads(q, q.shape[1], cache.head_dim, "queries")
    if q.get_device() != cache.device.index:
        raise ValueError(f"queries on {q.device}, the cache on {cache.device}")
    table = _index(table, torch.int32, 2, "table", cache.device)
    cu_q = _index(cu_q, torch.int32, 1, "cu_q", cache.device)
    kv_lens = _index(kv_lens, torch.int32, 1, "kv_lens", cache.device)
    (T, heads, dim), (B, width) = q.shape, table.shape
    if cu_q.shape[0] != B + 1 or kv_lens.shape[0] != B:
        raise ValueError(f"cu_q has {cu_q.shape[0]} and kv_lens {kv_lens.shape[0]} entries for "
                         f"{B} sequences")
    max_q = T if max_q is None else max(0, min(int(max_q), T))
    room = width * cache.page_size
    max_kv = room if max_kv is None else max(0, min(int(max_kv), room))
    out = q.new_empty((T, heads, dim))
    need = _lib.workspace_fast("paged_attention_workspace", T, heads, cache.kv_heads, dim, B,
                               max_q, max_kv)
    ws = _lib.scratch(need, q.device) if need else None
    q_token, q_head, _ = q.stride()
    _lib.call_fast("paged_attention", _lib.current_stream(), cache._address, q.data_ptr(),
                   q_token, q_head, _DTYPE_CODE[q.dtype], T, heads, table.data_ptr(),
                   max(table.stride(0), width), B, width, cu_q.data_ptr(), kv_lens.data_ptr(),
                   max_q, max_kv, 1.0 / math.sqrt(dim) if scale is None else float(scale),
                   out.data_ptr(), None if ws is None else ws.data_ptr(), need)
    return out
