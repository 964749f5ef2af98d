"""A cache in pages of 4-bit elements for several sequences: the pool, the tables, and their bookkeeping on the device.

    cache = PagedCache.allocate(n_pages=4096, n_slots=64, max_tokens=8192, n_kv_heads=8, head_dim=128, n_layers=32)
    cache.reserve(slots, counts)          room for counts[i] further tokens of sequence slots[i]
    ops.paged_kv_write(cache, k, v, ...)  per layer: the new tokens' keys and values
    ops.paged_attention(cache, q, ...)    per layer: the new tokens' attention
    cache.fork(src, dst)                  empty slots dst[i] continue sequences src[i]; pages are shared until one of them writes
    cache.free(slots)                     the sequences end
    cache.compact()                       the pages in use move to the pool's beginning

Every call runs on the current stream and reads its slots and counts from device memory: int32 tensors there, which a recorded
call reads anew, or lists, which are copied first (the copy waits for the stream, and cannot be recorded).  With tensors no call waits for
the device.  What a call finds wrong on the device is in `status`, which check() reads."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from . import ops


class PagedCache:
    """Views of one pool's tensors; `allocate` makes them.  pages: uint8 [n_pages, page_bytes], of every layer the part layer_bytes() (a
    view of some of the layers serves ops.paged_*, but no call that copies or moves pages: those take pages whole);
    tables: int32 [slots, most pages of a sequence], -1 behind a sequence's pages; lengths: int32 [slots]; refs: int32 [n_pages], how
    many slots hold a page."""

    def __init__(self, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, *, page_tokens: int = 64,
                 n_kv_heads: int = 1, head_dim: int = 0, status: torch.Tensor | None = None):
        for t, kind, dims in ((pages, torch.uint8, 2), (tables, torch.int32, 2), (lengths, torch.int32, 1), (refs, torch.int32, 1)):
            if t.dtype != kind or t.dim() != dims or not (t.is_contiguous() or t.stride(-1) == 1):
                raise RuntimeError("PagedCache: pages are uint8 [n, bytes], tables int32 [slots, n], lengths and refs int32 vectors, all with unit strides")
        if tables.shape[0] != lengths.shape[0] or refs.shape[0] != pages.shape[0] or pages.stride(0) % 16:
            raise RuntimeError("PagedCache: a length per table row, a count per page, pages on multiples of 16 bytes")
        if tables.shape[0] > 1 and tables.stride(0) != tables.shape[1]:  # (what bounds a sequence is the distance between two tables)
            raise RuntimeError("PagedCache: tables lie one behind the other; these are parts of wider ones")
        self.pages, self.tables, self.lengths, self.refs = pages, tables, lengths, refs
        self.page_tokens, self.n_kv_heads, self.head_dim, self.status = page_tokens, n_kv_heads, head_dim, status

    @classmethod
    def allocate(cls, n_pages: int, n_slots: int, max_tokens: int, n_kv_heads: int, head_dim: int, n_layers: int = 1, page_tokens: int = 64,
                 device: torch.device | str = "cuda") -> "PagedCache":
        layer = int(L.lib().cutb_paged_layer_bytes(n_kv_heads, head_dim, page_tokens))
        if layer == 0 or min(n_pages, n_slots, max_tokens, n_layers) < 1:
            raise ValueError("a page holds 16, 32, 64, 128 or 256 tokens, a head 1 .. 256 elements, and nothing is empty")
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        tables = i32(n_slots, -(-max_tokens // page_tokens)).fill_(-1)
        return cls(torch.zeros((n_pages, layer * n_layers), dtype=torch.uint8, device=device), tables, i32(n_slots), i32(n_pages),
                   page_tokens=page_tokens, n_kv_heads=n_kv_heads, head_dim=head_dim, status=i32(1))

    def layer_bytes(self) -> int:
        return int(L.lib().cutb_paged_layer_bytes(self.n_kv_heads, self.head_dim, self.page_tokens))

    def check(self) -> None:
        """Waits for the device; raises what a call has found wrong there since the last check."""
        st = int(self.status.item())
        if st:
            self.status.zero_()
            raise L.CutbError(st, L.lib().cutb_status_string(st).decode())

    # -- bookkeeping ------------------------------------------------------------------------------------------------
    def _vector(self, v, n: int | None = None) -> torch.Tensor:
        if not isinstance(v, torch.Tensor):
            v = torch.tensor([int(x) for x in v], dtype=torch.int32).to(self.tables.device)
        if v.dtype != torch.int32 or v.dim() != 1 or not v.is_contiguous() or v.get_device() != self.tables.get_device() or (n is not None and v.numel() != n):
            raise RuntimeError("slots, pages and counts are int32 vectors of one length on the device, or lists")
        return v

    def _desc(self, items=None, others=None, counts=None) -> "L.PagesDesc":
        d = L.PagesDesc()
        d.pages, d.page_bytes, d.ld_table = self.pages.data_ptr(), self.pages.shape[1], self.tables.shape[1]
        d.n_pages, d.page_tokens, d.n_slots = self.pages.shape[0], self.page_tokens, self.tables.shape[0]
        d.tables, d.lengths, d.refs = self.tables.data_ptr(), self.lengths.data_ptr(), self.refs.data_ptr()
        if items is not None:
            d.n, d.items, d.others, d.counts = items.numel(), items.data_ptr(), ops._ptr(others), ops._ptr(counts)
        d.status = ops._ptr(self.status)
        return d

    def _whole(self, what: str) -> None:
        """Pages are copied from one place of the pool to the next one's, which must not be more than this cache's."""
        if self.pages.shape[0] > 1 and self.pages.stride(0) != self.pages.shape[1]:
            raise RuntimeError(f"{what}: pages are moved whole, and these are parts of wider ones")

    def _run(self, name: str, d, workspace: bool) -> None:
        ops._here(name, self.pages, self.tables, self.lengths, self.refs, self.status)
        if workspace:
            need = int(L.lib().cutb_pages_workspace_bytes(C.byref(d)))
            ws = self.pages.new_empty(need)
            d.workspace, d.workspace_bytes = ws.data_ptr(), need
        L.check(getattr(L.lib(), name)(C.byref(d), ops._stream_ptr()))

    def reserve(self, slots, counts) -> None:
        """Sequence slots[i] grows by counts[i] tokens, first come, first served, in whole entries: with too few free pages the entries
        from the first that does not fit on keep their lengths (CUTB_ERR_PAGES).  A shared last page is copied before it is written."""
        self._whole("reserve")
        slots = self._vector(slots)
        counts = self._vector(counts, slots.numel())
        self._run("cutb_pages_reserve", self._desc(slots, counts=counts), True)

    def fork(self, src, dst) -> None:
        src = self._vector(src)
        dst = self._vector(dst, src.numel())
        self._run("cutb_pages_fork", self._desc(src, dst), False)

    def free(self, slots) -> None:
        slots = self._vector(slots)
        self._run("cutb_pages_free", self._desc(slots), False)

    def compact(self) -> None:
        self._whole("compact")
        self._run("cutb_pages_compact", self._desc(), True)

    def copy(self, src, dst) -> None:
        """Page dst[i] becomes a copy of page src[i], every dst named once (tables and refs are the caller's)."""
        self._whole("copy")
        src = self._vector(src)
        dst = self._vector(dst, src.numel())
        self._run("cutb_pages_copy", self._desc(src, dst), False)
