"""Paged KV cache for the Qwen3 model: one page pool per layer, pages shared by
all requests, a host-side page list per request.

Follows the reference's ``TinyKvPagedPool`` / ``TinyKvPagedCache``
(``cache/paged.py:21-559``) and its per-layer pools (``models/qwen3.py:272-283``):
a pool holds ``key_pages``/``value_pages [P, num_kv_heads, page_size, D]``;
token ``j`` of a request lives in slot ``j % page_size`` of the request's page
``j // page_size``.  Here every pool is allocated once at its full size (HBM
is large) instead of grown geometrically, and one free list serves all layers
(a request holds the same page ids in every layer).  ``kv_bits`` 4 holds pages
in MXFP4 (``MxPages``, 4.25 bits a value; the reference's quantised cache has
eight).  Prefix caching and int8 pages are not built.
"""

from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

import torch

from .mx import MX_DTYPES, mx_quantize
from .mx_cache import MxPages, paged_kv_read_mx


class PagedKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 kv_bits: int = 16):
        if num_pages <= 0 or page_size <= 0:
            raise ValueError("PagedKVCache: num_pages and page_size must be positive")
        if kv_bits not in (4, 16):
            raise ValueError(f"PagedKVCache: kv_bits must be 4 or 16, got {kv_bits}")
        if kv_bits == 4 and (head_dim % 32 or not 0 < head_dim <= 256):
            raise ValueError(f"PagedKVCache: kv_bits=4 needs a head dim that is a multiple of 32, at "
                             f"most 256, got {head_dim}")
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.num_pages = num_pages
        self.page_size = page_size
        self.dtype = dtype
        self.kv_bits = kv_bits
        self.device = torch.device(device)
        # one page past the pool takes the writes of padding rows and of
        # graph warm-up/capture runs; it is never handed to a request
        self.scratch_page = num_pages
        shape = (num_pages + 1, num_kv_heads, page_size, head_dim)

        def pool():
            if kv_bits == 4:
                return MxPages.zeros(*shape, device=self.device)
            return torch.zeros(shape, dtype=dtype, device=self.device)

        self.key_pages = [pool() for _ in range(num_layers)]
        self.value_pages = [pool() for _ in range(num_layers)]
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self.pages: Dict[int, List[int]] = {}
        self.lens: Dict[int, int] = {}

    # ---------------------------------------------------------------- requests

    def add(self, seq_id: int) -> None:
        if seq_id in self.pages:
            raise ValueError(f"sequence {seq_id} already has a cache")
        self.pages[seq_id] = []
        self.lens[seq_id] = 0

    def free(self, seq_id: int) -> None:
        """Return the request's pages to the pool."""
        self._free.extend(reversed(self.pages.pop(seq_id)))
        del self.lens[seq_id]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_needed(self, seq_id: int, n_new: int) -> int:
        total = self.lens[seq_id] + n_new
        return max(0, -(-total // self.page_size) - len(self.pages[seq_id]))

    def reserve(self, seq_id: int, n_new: int) -> None:
        """Make room for ``n_new`` more tokens of the request."""
        need = self.pages_needed(seq_id, n_new)
        if need > len(self._free):
            raise RuntimeError(f"PagedKVCache: out of pages ({need} needed, "
                               f"{len(self._free)} free)")
        for _ in range(need):
            self.pages[seq_id].append(self._free.pop())

    # ---------------------------------------------------------------- one step

    def slot_mapping(self, seq_ids: Sequence[int], n_new: int):
        """(page ids, slots) of the next ``n_new`` tokens of every request, in
        request-major order, as device tensors (after ``reserve``)."""
        pages, slots = [], []
        ps = self.page_size
        for s in seq_ids:
            plist, start = self.pages[s], self.lens[s]
            for j in range(start, start + n_new):
                pages.append(plist[j // ps])
                slots.append(j % ps)
        dev = self.device
        return (torch.tensor(pages, dtype=torch.int32, device=dev),
                torch.tensor(slots, dtype=torch.int32, device=dev))

    def _mapped(self, page_ids: torch.Tensor, slots: torch.Tensor):
        """Which slots exist, and 64-bit indices of theirs (0 for others): indexing
        out of bounds would end the process, and below zero it counts from the end."""
        page_ids, slots = page_ids.long(), slots.long()
        there = ((page_ids >= 0) & (page_ids <= self.num_pages) & (slots >= 0)
                 & (slots < self.page_size))
        return there, page_ids * there, slots * there

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, page_ids: torch.Tensor,
              slots: torch.Tensor) -> None:
        """Store ``k``/``v [B, L, num_kv_heads, D]`` at the mapped slots (for
        callers that compute k/v themselves; the model's fused q/k kernel
        stores them directly).  Four bits are taken of the values as they come,
        without a rounding to the cache's dtype before it (of float64 ones as
        float32).  Slots outside the pages are not stored (their values go to the
        scratch page)."""
        there, page_ids, slots = self._mapped(page_ids, slots)
        page_ids = torch.where(there, page_ids, self.scratch_page)
        for pages, x in ((self.key_pages[layer], k), (self.value_pages[layer], v)):
            x = x.reshape(-1, self.num_kv_heads, self.head_dim)
            if self.kv_bits == 4:
                t = mx_quantize(x if x.dtype in MX_DTYPES else x.float(), "mxfp4")
                pages.codes[page_ids, :, slots] = t.codes
                pages.scales[page_ids, :, slots] = t.scales
            else:
                pages[page_ids, :, slots, :] = x.to(self.dtype)

    def read(self, layer: int, page_ids: torch.Tensor, slots: torch.Tensor
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """What the mapped slots hold: ``k, v [T, num_kv_heads, D]`` of the
        cache's dtype.  Slots outside the pages give zeros."""
        kp, vp = self.key_pages[layer], self.value_pages[layer]
        if self.kv_bits == 4:
            return paged_kv_read_mx(kp, vp, page_ids, slots, self.dtype)
        there, page_ids, slots = self._mapped(page_ids, slots)
        gone = ~there[:, None, None]
        return tuple(pages[page_ids, :, slots, :].masked_fill(gone, 0) for pages in (kp, vp))

    def advance(self, seq_ids: Sequence[int], n_new: int) -> None:
        for s in seq_ids:
            self.lens[s] += n_new

    def block_table(self, seq_ids: Sequence[int], extra: int = 0, width: int | None = None):
        """``block_table [B, width]`` (-1 past a request's pages; width defaults
        to the longest page list) and ``context_lens [B]`` (current length +
        ``extra``) as int32 tensors."""
        width = width or max(1, max(len(self.pages[s]) for s in seq_ids))
        rows = [self.pages[s] + [-1] * (width - len(self.pages[s])) for s in seq_ids]
        dev = self.device
        return (torch.tensor(rows, dtype=torch.int32, device=dev),
                torch.tensor([self.lens[s] + extra for s in seq_ids], dtype=torch.int32,
                             device=dev))
