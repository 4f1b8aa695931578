"""Page tables and slot maps of a ``PagedKVCache``, kept on the GPU.

Every request has a row of page numbers and a length; free pages lie on a stack.  A step of a
batch takes the pages that its new tokens need and gives what the cache's calls ask for:

    tables = PageTables(cache.num_pages, cache.page_size, max_seqs=64, max_pages=128)
    step = tables.extend(rows, new, total)          # rows and counts of this step's requests
    cache.write(k, v, step.slots)
    out = paged_attention(q, cache, step.table, step.cu, step.kv_lens)
    tables.release(rows)                            # requests that are done

Nothing waits for the GPU, and a step can be captured into a graph, each replay of which takes
its own pages.  Requests that cannot be placed are left as they were and flagged;
``tables.check()`` raises for them at a point of the caller's choosing.
"""
import ctypes
from collections import namedtuple

import torch

from . import _lib

PageStep = namedtuple("PageStep", "table cu kv_lens slots positions")
_I32, _I64 = torch.int32, torch.int64


class PageTables:
    """Rows for ``max_seqs`` requests of up to ``max_pages`` pages each, over the
    ``num_pages`` pages of ``page_size`` slots of a cache.

    ``table`` (max_seqs, max_pages) int32 holds page numbers and −1 where there is none,
    ``lengths`` (max_seqs,) int32 the requests' tokens; ``free_pages[:free_count]`` is the stack
    of free pages, the last on top (at first page 0).  Calls on one ``PageTables`` change these
    and have to follow each other on one stream."""

    def __init__(self, num_pages, page_size, max_seqs, max_pages, device="cuda"):
        if page_size < 1 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"PageTables: pages of {page_size} slots (a power of two up to 4096 "
                             "is needed)")
        if not 0 <= num_pages < 1 << 31 or not 1 <= max_seqs < 1 << 31 or max_pages < 1 \
                or max_pages * page_size >= 1 << 31:
            raise ValueError(f"PageTables: {max_seqs} rows of {max_pages} of {num_pages} pages "
                             "(fewer than 2^31 slots in a row)")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("PageTables live on the GPU")
        self.num_pages, self.page_size = num_pages, page_size
        self.max_seqs, self.max_pages = max_seqs, max_pages
        i32 = dict(dtype=_I32, device=dev)
        self._held = (torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(max_seqs, **i32),
                      torch.arange(num_pages - 1, -1, -1, **i32),
                      torch.full((1,), num_pages, **i32),
                      torch.full((max_seqs,), 0x7fffffff, **i32), torch.zeros(1, **i32))
        self.device = self._held[0].device
        self._device = self.device.index
        self._struct = _lib.PageTablesStruct(*(_lib.ptr(t) if t.numel() else None
                                               for t in self._held),
                                             max_seqs, max_pages, num_pages, page_size)
        self._address = ctypes.addressof(self._struct)

    # (the kernels know these by their addresses: changed in place, never replaced)
    table, lengths, free_pages, free_count, _mark, flags = (
        property(lambda self, i=i: self._held[i]) for i in range(6))

    def _index(self, t, what, like=None):
        if t.dim() != 1 or t.dtype is not _I32:
            raise ValueError(f"PageTables: {what} of {t.dtype} and shape {tuple(t.shape)} (int32, "
                             "one per request)")
        if t.get_device() != self._device:
            raise ValueError(f"PageTables: {what} on {t.device}, the tables on {self.device}")
        if torch._C._cuda_getDevice() != self._device:
            raise ValueError(f"PageTables on {self.device} while device "
                             f"{torch._C._cuda_getDevice()} is current")
        if like is not None and t.shape != like.shape:
            raise ValueError(f"PageTables: {len(like)} rows, {len(t)} {what}")
        if len(t) > 1 << 20:
            raise ValueError(f"PageTables: {len(t)} requests in one call (at most 2^20)")
        return t if t.is_contiguous() else t.contiguous()

    def extend(self, rows, new, total):
        """Room for ``new[i]`` more tokens of the request in row ``rows[i]`` (both int32 on the
        GPU, a row at most once): ``(table, cu, kv_lens, slots, positions)``.

        ``total`` is the number of tokens of the step, or more where it is padded.  ``table``
        (B, max_pages), ``cu`` (B + 1) and ``kv_lens`` (B) int32 are the batch's page tables,
        token offsets and lengths with the new tokens, as ``paged_attention`` takes them;
        ``slots`` and ``positions`` (total,) int64 say where each token goes (slot −1 and
        position 0 for padding and for tokens that were not placed).

        Negative rows are padding.  A request is left as it was and its tokens are not placed
        (they keep their places in ``cu``) where the free pages or its row do not suffice, in
        the order of the batch, and where its row is none, came before in the batch, or its
        tokens end past ``total``."""
        # what is usual passes in one go (a call is a few microseconds); the rest is told apart
        if not (rows.dtype is new.dtype is _I32 and rows.dim() == 1 and rows.shape == new.shape
                and rows.is_contiguous() and new.is_contiguous() and rows.shape[0] <= 1 << 20
                and rows.get_device() == new.get_device() == self._device
                and torch._C._cuda_getDevice() == self._device):
            rows = self._index(rows, "rows")
            new = self._index(new, "counts", rows)
        B, total, width, dev = rows.shape[0], int(total), self.max_pages, self.device
        if not 0 <= total < 1 << 31:
            raise ValueError(f"PageTables: a step of {total} tokens")
        # the workspace lies behind the offsets and lengths
        need = _lib.workspace_fast("pages_workspace", B)
        table = torch.empty(B, width, dtype=_I32, device=dev)
        small = torch.empty(2 * B + 1 + need // 4, dtype=_I32, device=dev)
        slots, positions = torch.empty(2, total, dtype=_I64, device=dev).unbind()
        cu, kv_lens, _ = small.split_with_sizes((B + 1, B, need // 4))
        at = small.data_ptr()
        _lib.call_fast("pages_extend", _lib.current_stream(), self._address, rows.data_ptr(),
                       new.data_ptr(), B, total, table.data_ptr(), at, at + 4 * (B + 1),
                       slots.data_ptr(), positions.data_ptr(), at + 4 * (2 * B + 1), need)
        return PageStep(table, cu, kv_lens, slots, positions)

    def release(self, rows, keep=None):
        """Cut the requests in ``rows`` (int32) to their first ``keep[i]`` tokens (int32; None:
        none) and give their other pages back.  Releasing what one ``extend`` took, with the same
        rows, leaves the stack as it was.  ``keep`` outside 0 to the request's length changes
        nothing and is flagged, as are rows that are none or come twice; negative rows are
        padding."""
        if not (rows.dtype is _I32 and rows.dim() == 1 and rows.is_contiguous()
                and rows.shape[0] <= 1 << 20
                and (keep is None or (keep.dtype is _I32 and keep.shape == rows.shape
                                      and keep.is_contiguous()
                                      and keep.get_device() == self._device))
                and rows.get_device() == torch._C._cuda_getDevice() == self._device):
            rows = self._index(rows, "rows")
            keep = None if keep is None else self._index(keep, "counts", rows)
        B = rows.shape[0]
        if B:
            need = _lib.workspace_fast("pages_workspace", B)
            ws = _lib.scratch(need, self.device)
            _lib.call_fast("pages_release", _lib.current_stream(), self._address, rows.data_ptr(),
                           None if keep is None else keep.data_ptr(), B, ws.data_ptr(), need)

    def check(self):
        """Raise if a request could not be placed, or a row or count was none, since the last
        check (waits for the current stream): IndexError for the latter, also where both were met
        (its message then names both), else RuntimeError."""
        v = int(self.flags.item())
        self.flags.zero_()
        room = "no free page, or a request longer than its row"
        if v & _lib.FLAG_BAD_INDEX:
            raise IndexError("PageTables: a row outside the tables or given twice, a count out of "
                             "range, or more tokens than the step's total"
                             + (f"; and {room}" if v & _lib.FLAG_NO_ROOM else ""))
        if v & _lib.FLAG_NO_ROOM:
            raise RuntimeError(f"PageTables: {room}")
