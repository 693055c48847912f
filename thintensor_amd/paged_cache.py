"""The paged KV cache in 16 bits that ``rotary_append_paged``, ``gqa_attention_paged`` and
``select_pages`` of :class:`~thintensor_amd.backend.HipDecodeBackend` work on.

* ``k_pages``, ``v_pages`` fp16 or bf16 [pages, kv_heads, page_size, head_dim];
* ``k_bounds`` (optional, for ``select_pages``) of the same type [pages, kv_heads, 2, head_dim]: of every
  dim the least and the greatest key of a page.

Token t of a row lies in page ``page_table[row, t // page_size]``, slot ``t % page_size``; which pages
belong to whom is the caller's bookkeeping, and rows may share pages that hold the same tokens.  Strides of
pages, heads and tokens are free, so a cache laid out [pages, page_size, kv_heads, head_dim] or with
K and V side by side comes in as a view.  Contents past a row's length are never used.
"""

from __future__ import annotations

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class PagedKvCache:
    """Tensors of a paged KV cache and the descriptor that the kernels take."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, k_bounds: torch.Tensor | None = None) -> None:
        if k_pages.ndim != 4 or v_pages.shape != k_pages.shape:
            raise ValueError("paged cache takes k_pages and v_pages [pages, kv_heads, page_size, head_dim]")
        if k_pages.dtype not in _DTYPES or v_pages.dtype != k_pages.dtype:
            raise ValueError("paged cache tensors must be float16 or bfloat16, of one type")
        pages, kv_heads, page_size, head_dim = map(int, k_pages.shape)
        if pages < 1 or kv_heads < 1:
            raise ValueError("paged cache needs at least one page and KV head")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"paged cache head_dim must be 64, 128 or 256, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"paged cache page_size must be 16, 32, 64, 128 or 256, got {page_size}")
        if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
            raise ValueError("paged cache tensors must be contiguous in their last axis")
        if k_bounds is not None:
            if tuple(k_bounds.shape) != (pages, kv_heads, 2, head_dim) or k_bounds.dtype != k_pages.dtype:
                raise ValueError("paged cache k_bounds must be [pages, kv_heads, 2, head_dim] of the pages' type")
            if k_bounds.stride(3) != 1 or k_bounds.stride(2) != head_dim:
                raise ValueError("paged cache k_bounds must be contiguous in their last two axes")
        tensors = (k_pages, v_pages) if k_bounds is None else (k_pages, v_pages, k_bounds)
        if len({t.device for t in tensors}) != 1:
            raise ValueError("paged cache tensors must be on one device")
        self._tensors = k_pages, v_pages, k_bounds         # the descriptor holds their addresses: they stay
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, head_dim
        self.dtype, self.device = k_pages.dtype, k_pages.device
        ks, vs, bs = k_pages.stride(), v_pages.stride(), (0, 0) if k_bounds is None else k_bounds.stride()
        self.desc = _lib.PagedCache(
            k_pages.data_ptr(), v_pages.data_ptr(), None if k_bounds is None else k_bounds.data_ptr(),
            ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], bs[0], bs[1], pages, kv_heads, page_size, head_dim,
            _DTYPES[self.dtype])

    @property
    def k_pages(self) -> torch.Tensor:
        return self._tensors[0]

    @property
    def v_pages(self) -> torch.Tensor:
        return self._tensors[1]

    @property
    def k_bounds(self) -> torch.Tensor | None:
        return self._tensors[2]

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.float16, *,
                 bounds: bool = False, device: torch.device | str = "cuda") -> "PagedKvCache":
        """A cache of zeros, with ``k_bounds`` if asked for."""
        if pages < 1 or kv_heads < 1:
            raise ValueError("paged cache needs at least one page and KV head")
        if head_dim not in (64, 128, 256) or page_size not in PAGE_SIZES:
            raise ValueError("paged cache head_dim must be 64, 128 or 256 and page_size 16, 32, 64, 128 or 256")
        zeros = lambda *shape: torch.zeros(shape, device=device, dtype=dtype)  # noqa: E731
        return cls(zeros(pages, kv_heads, page_size, head_dim), zeros(pages, kv_heads, page_size, head_dim),
                   zeros(pages, kv_heads, 2, head_dim) if bounds else None)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._tensors if t is not None)
