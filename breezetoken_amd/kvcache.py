"""Fixed-capacity bf16 KV cache laid out for gfx950 HBM3E.

Mirrors the reference ``KVCache`` (breezetoken/model/config.py:100-111): one
layer's ``k`` and ``v`` are ``(max_context, n_kv * head_dim)`` tensors, token
major, so every caller view keeps working unchanged:

* ``cache.k[pos] = k.reshape(-1)``                  (layers.py:71-73)
* ``cache.k[:seq].view(seq, n_kv, head_dim)``       (layers.py:77-78)
* ``cache.k.index_copy_(0, index, k.reshape(1, -1))`` (graph.py:52-53)
* ``cache.k.view(cap, n_kv, head_dim)``             (graph.py:57-58)
* ``cache.k[:steps] = k.reshape(steps, -1)``        (prefill.py:54-55)

Differences from the reference, all below the view contract:

* dtype is bf16 (the reference stores f32, config.py:104-106 with
  qwen35.py:118-121); writers must cast, e.g. ``index_copy_`` needs
  ``k.to(torch.bfloat16)``;
* ``k`` and ``v`` are prefix views of one allocation whose slot count is padded
  up to a multiple of ``SLOT_ALIGN`` (whole 32-token tiles) plus one spare tile,
  and whose base is 256-byte aligned, so the decode kernel's 16-byte loads of a
  partial last tile stay inside the allocation;
* K and V of one layer sit in one allocation (K first), so a layer's cache is a
  single HBM extent.

``PagedKVCache`` is the cache of many sequences at once, of every layer, in
pages: a page table names each sequence's pages, which sequences may share.
"""

from __future__ import annotations

import torch

PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)  # tokens; a 16-token decode tile never crosses a page
SLOT_ALIGN = 32  # the reference's K/V tile (cap % block_n == 0, attention.py:227-228): two 16-token decode tiles


def padded_slots(capacity: int) -> int:
    return -(-capacity // SLOT_ALIGN) * SLOT_ALIGN + SLOT_ALIGN


class KVCache:
    """One attention layer's bf16 KV cache: ``k``/``v`` are ``(capacity, n_kv*head_dim)``."""

    def __init__(
        self,
        capacity: int,
        n_kv: int,
        head_dim: int,
        device: str | torch.device,
        dtype: torch.dtype = torch.bfloat16,
    ) -> None:
        if capacity <= 0 or n_kv <= 0 or head_dim <= 0:
            raise ValueError("capacity, n_kv and head_dim must be positive")
        if dtype != torch.bfloat16:
            raise ValueError("the MI355X cache is bf16")
        self.capacity = capacity
        self.n_kv = n_kv
        self.head_dim = head_dim
        row = n_kv * head_dim
        slots = padded_slots(capacity)
        self._store = torch.zeros((2, slots, row), device=device, dtype=dtype)
        if self._store.is_cuda and self._store.data_ptr() % 256:
            raise RuntimeError("cache allocation is not 256-byte aligned")
        self.k = self._store[0, :capacity]
        self.v = self._store[1, :capacity]

    @property
    def device(self) -> torch.device:
        return self._store.device

    def views(self) -> tuple[torch.Tensor, torch.Tensor]:
        """``(capacity, n_kv, head_dim)`` views, as the graph path passes them (graph.py:57-58)."""
        shape = (self.capacity, self.n_kv, self.head_dim)
        return self.k.view(shape), self.v.view(shape)

    def reset(self) -> None:
        # Slots are written before they are read (config.py:108-111); nothing to clear.
        pass

    def nbytes(self) -> int:
        return self._store.numel() * self._store.element_size()


class PagedKVCache:
    """The bf16 KV cache of ``layers`` attention layers in ``num_pages`` pages of
    ``page_size`` tokens; a page id names that page of every layer's K and V.

    * ``layer(i)``: layer i's ``k``/``v`` as (num_pages, page_size, n_kv, head_dim)
      views, what ``HipBackend.attn_prep_paged`` and ``attention_paged`` take;
    * ``pages``: all of it as (2 * layers, num_pages, page_size, n_kv * head_dim),
      what ``fork_pages`` and ``compact_pages`` take;
    * ``rows(i, first, count)``: the tokens of consecutive pages as the flat (count,
      n_kv, head_dim) rows that ``attention_prefill`` reads.  ``fork_pages`` gives
      free pages lowest first, so after ``compact_pages`` (or in a fresh cache) a
      prompt's pages are consecutive.

    The page table (rows, P) int32 and the lengths (rows,) int32 are plain device
    tensors; ``empty_table`` makes those of rows without tokens."""

    def __init__(self, num_pages: int, page_size: int, n_kv: int, head_dim: int, device: str | torch.device,
                 layers: int = 1) -> None:
        if num_pages <= 0 or n_kv <= 0 or head_dim <= 0 or layers <= 0:
            raise ValueError("num_pages, n_kv, head_dim and layers must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if n_kv * head_dim % 8:
            raise ValueError("n_kv * head_dim must be a multiple of 8")
        self.num_pages, self.page_size, self.layers = num_pages, page_size, layers
        self.n_kv, self.head_dim = n_kv, head_dim
        self.pages = torch.zeros((2 * layers, num_pages, page_size, n_kv * head_dim), dtype=torch.bfloat16, device=device)

    @property
    def device(self) -> torch.device:
        return self.pages.device

    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        if not 0 <= i < self.layers:
            raise IndexError(f"layer {i} of {self.layers}")
        shape = (self.num_pages, self.page_size, self.n_kv, self.head_dim)
        return self.pages[2 * i].view(shape), self.pages[2 * i + 1].view(shape)

    def rows(self, i: int, first: int, count: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Layer i's first ``count`` tokens from page ``first`` on, over consecutive pages."""
        at = first * self.page_size
        if first < 0 or count < 0 or at + count > self.num_pages * self.page_size:
            raise IndexError("rows outside the cache")
        k, v = self.layer(i)
        flat = (-1, self.n_kv, self.head_dim)
        return k.view(flat)[at : at + count], v.view(flat)[at : at + count]

    def empty_table(self, rows: int, max_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(table, lens) of ``rows`` sequences without tokens, of up to ``max_tokens`` each."""
        if rows < 0 or max_tokens <= 0:
            raise ValueError("rows must not be negative, max_tokens must be positive")
        table = torch.full((rows, -(-max_tokens // self.page_size)), -1, dtype=torch.int32, device=self.device)
        return table, torch.zeros(rows, dtype=torch.int32, device=self.device)

    def nbytes(self) -> int:
        return self.pages.numel() * self.pages.element_size()
