"""The KV cache of 4 bits that ``kv_append_int4``, ``kv_read_int4`` and ``gqa_attention_int4`` of
:class:`~thintensor_amd.backend.HipDecodeBackend` work on.

Groups of 32, 64 or 128 dims of one token and KV head share a step and a minimum in fp16; a value
is code x step + minimum with a code of 4 bits.  Per token and KV head it takes
head_dim + 8 head_dim / group_size bytes for K and V together, against 4 head_dim in 16 bits.

* ``k_codes`` int32 [batch, kv_heads, capacity, head_dim / 8]: dim d in nibble d % 8 of word d / 8;
* ``k_scales`` fp16 [batch, kv_heads, capacity, groups, 2]: (step, minimum);
* ``v_codes`` int32 [batch, kv_heads, capacity / 8, head_dim]: token t of a block of eight in nibble
  t / 2 + 4 (t % 2) of the dim's word, so that the product with V reads tokens together;
* ``v_scales`` fp16 [batch, kv_heads, capacity / 8, groups, 2, 8]: eight steps, eight minima.

Contents past a sequence's length are never used, so a cache need not be cleared.
"""

from __future__ import annotations

import torch

from . import _lib


class Int4KvCache:
    """Tensors of a 4-bit KV cache and the descriptor that the kernels take."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                 v_scales: torch.Tensor) -> None:
        if k_codes.ndim != 4 or k_scales.ndim != 5 or v_codes.ndim != 4 or v_scales.ndim != 6:
            raise ValueError("4-bit cache tensors must have ranks 4, 5, 4 and 6")
        if k_codes.dtype != torch.int32 or v_codes.dtype != torch.int32 or k_scales.dtype != torch.float16 or \
                v_scales.dtype != torch.float16:
            raise ValueError("4-bit cache codes must be int32 and scales float16")
        batch, kv_heads, capacity, words = map(int, k_codes.shape)
        head_dim, groups = 8 * words, int(k_scales.shape[3])
        if batch < 1 or kv_heads < 1:
            raise ValueError("4-bit cache needs at least one sequence and KV head")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"4-bit cache head_dim must be 64, 128 or 256, got {head_dim}")
        if groups < 1 or head_dim % groups or head_dim // groups not in (32, 64, 128):
            raise ValueError("4-bit cache groups must be of 32, 64 or 128 dims")
        if capacity < 1 or capacity % 32:
            raise ValueError(f"4-bit cache capacity must be a multiple of 32 tokens, got {capacity}")
        if tuple(k_scales.shape) != (batch, kv_heads, capacity, groups, 2) or \
                tuple(v_codes.shape) != (batch, kv_heads, capacity // 8, head_dim) or \
                tuple(v_scales.shape) != (batch, kv_heads, capacity // 8, groups, 2, 8):
            raise ValueError("4-bit cache tensors do not match each other")
        if len({t.device for t in (k_codes, k_scales, v_codes, v_scales)}) != 1:
            raise ValueError("4-bit cache tensors must be on one device")
        for t in (k_codes, k_scales, v_codes, v_scales):
            if not t[0, 0].is_contiguous():
                raise ValueError("4-bit cache tensors must be contiguous within a sequence and head")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.batch, self.kv_heads, self.capacity, self.head_dim = batch, kv_heads, capacity, head_dim
        self.group_size = head_dim // groups
        self.device = k_codes.device
        self.desc = _lib.Int4Cache(
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
            k_codes.stride(0), k_codes.stride(1), k_scales.stride(0), k_scales.stride(1),
            v_codes.stride(0), v_codes.stride(1), v_scales.stride(0), v_scales.stride(1),
            batch, kv_heads, capacity, head_dim, self.group_size)

    @classmethod
    def allocate(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, group_size: int = 32,
                 device: torch.device | str = "cuda") -> "Int4KvCache":
        """An empty cache; the capacity is rounded up to whole blocks of 32 tokens."""
        if group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError("4-bit cache groups must be of 32, 64 or 128 dims and at most head_dim")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"4-bit cache head_dim must be 64, 128 or 256, got {head_dim}")
        if batch < 1 or kv_heads < 1 or capacity < 1:
            raise ValueError("4-bit cache needs at least one sequence, KV head and token")
        cap, groups = -(-capacity // 32) * 32, head_dim // group_size
        return cls(torch.zeros((batch, kv_heads, cap, head_dim // 8), device=device, dtype=torch.int32),
                   torch.zeros((batch, kv_heads, cap, groups, 2), device=device, dtype=torch.float16),
                   torch.zeros((batch, kv_heads, cap // 8, head_dim), device=device, dtype=torch.int32),
                   torch.zeros((batch, kv_heads, cap // 8, groups, 2, 8), device=device, dtype=torch.float16))

    def sequences(self, start: int, stop: int) -> "Int4KvCache":
        """Sequences start .. stop - 1 of this cache, as a view."""
        if not 0 <= start < stop <= self.batch:
            raise ValueError(f"sequences {start} .. {stop} of a cache of {self.batch}")
        return Int4KvCache(self.k_codes[start:stop], self.k_scales[start:stop], self.v_codes[start:stop],
                           self.v_scales[start:stop])

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales))
