"""Paged 8-bit KV caches: the page pool and the batch plan of `Engine.paged_append` and
`Engine.paged_attention` (the reference's caches are one contiguous buffer per request).

    cache = eng.new_paged_cache(pages, page_size=32)
    pool = PagedPool(cache)                                   # free pages; pool.grow / release / table
    plan = eng.paged_plan(rows, start, page_size=32)          # one per step, shared by every layer
    q = eng.paged_append(cache, layer, plan, table, q, k, v)  # rotate, code, write
    o = eng.paged_attention(cache, layer, plan, table, q)
"""

from __future__ import annotations

import ctypes
import dataclasses

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)


@dataclasses.dataclass(frozen=True, eq=False)
class PagedCache:
    """A pool of pages: float8 e4m3 codes [layers, pages, kv_heads, page_size, head_dim] of the keys
    and of the values, and fp32 scales [layers, pages, kv_heads]; a cached value is code * scale.
    Immutable (its tensors' contents are not), so that it is checked once, not in every layer's call."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        if self.k.dim() != 5 or self.k.shape != self.v.shape:
            raise ValueError("paged cache: k and v must be [layers, pages, kv_heads, page_size, head_dim]")
        if self.k.shape[3] not in PAGE_SIZES:
            raise ValueError(f"paged cache: page size must be one of {PAGE_SIZES}, got {self.k.shape[3]}")
        for t in (self.k, self.v):
            if t.dtype != torch.float8_e4m3fn or not t.is_contiguous():
                raise ValueError("paged cache: codes must be contiguous float8_e4m3fn")
        for t in (self.k_scale, self.v_scale):
            if t.dtype != torch.float32 or not t.is_contiguous() or t.shape != self.k.shape[:3]:
                raise ValueError("paged cache: scales must be contiguous float32 [layers, pages, kv_heads]")
        if len({t.device for t in (self.k, self.v, self.k_scale, self.v_scale)}) != 1:
            raise ValueError("paged cache: tensors on different devices")
        desc = _lib.FdllmPagedCache(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                                    self.v_scale.data_ptr(), self.layers, self.pages, self.page_size)
        object.__setattr__(self, "device", self.k.device)
        object.__setattr__(self, "heads", (int(self.k.shape[2]), int(self.k.shape[4])))  # KV heads, head dim
        object.__setattr__(self, "_desc", desc)
        object.__setattr__(self, "ref", ctypes.byref(desc))

    @property
    def layers(self) -> int:
        return int(self.k.shape[0])

    @property
    def pages(self) -> int:
        return int(self.k.shape[1])

    @property
    def page_size(self) -> int:
        return int(self.k.shape[3])


class PagedPool:
    """The free pages of a cache.  Requests take pages as they grow and give them back when done."""

    def __init__(self, cache: PagedCache):
        self.cache = cache
        self._free = list(range(cache.pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def grow(self, pages: list[int], rows: int) -> None:
        """Extend a request's page list to hold `rows` cache rows."""
        need = -(-rows // self.cache.page_size) - len(pages)
        if need > len(self._free):
            raise MemoryError(f"paged cache: {need} pages needed, {len(self._free)} free")
        pages.extend(self._free.pop() for _ in range(need))

    def release(self, pages: list[int]) -> None:
        self._free.extend(reversed(pages))
        pages.clear()

    def table(self, requests: list[list[int]]) -> torch.Tensor:
        """int32 [n, columns] page table of several requests on the cache's device."""
        width = max((len(p) for p in requests), default=0) or 1
        host = torch.zeros((len(requests), width), dtype=torch.int32, pin_memory=self.cache.device.type == "cuda")
        rows = host.numpy()
        for i, p in enumerate(requests):
            rows[i, :len(p)] = p
        return host.to(self.cache.device, non_blocking=True)


class PagedPlan:
    """A laid-out batch (fdllm_paged_plan_batch): the host description and its words on the device.
    `words` is read by the calls that take the plan, in stream order after its upload."""

    def __init__(self, desc, words: torch.Tensor, staging: torch.Tensor):
        self.desc = desc
        self.words = words
        self._staging = staging  # pinned source of the upload, alive as long as the plan
        self.ref = ctypes.byref(desc)
        self.words_ptr = words.data_ptr()
        self.device = words.device
        self.n = int(desc.n)
        self.total_rows = int(desc.total_rows)
        self.table_cols = int(desc.table_cols)  # columns a page table needs
