"""Layouts of outputs that share no memory though they lie in one buffer."""

from __future__ import annotations

import pytest
import torch

from thintensor_amd.kv_cache import Int4KvCache

pytestmark = pytest.mark.gpu


def _held(backend, device, batch, kv_heads, capacity, dim):
    g = torch.Generator(device=device).manual_seed(dim)
    cache = Int4KvCache.allocate(batch, kv_heads, capacity, dim, 32, device)
    k, v = (torch.randn((batch, capacity, kv_heads, dim), generator=g, device=device).half() for _ in range(2))
    backend.kv_append_int4(cache, k, v, torch.zeros(batch, device=device, dtype=torch.int32))
    return cache, g


def test_read_into_parts_of_one_buffer(backend, device):
    """K and V side by side in a row, head by head, tokens or heads as the slowest axis."""
    cache, _ = _held(backend, device, 3, 2, 32, 64)
    starts = torch.tensor([0, 3, 9], device=device, dtype=torch.int32)
    want = backend.kv_read_int4(cache, *(torch.empty((3, 5, 2, 64), device=device).half() for _ in range(2)), starts)
    buffers = []
    rows = torch.full((3, 5, 4, 64), 7.0, device=device).half()
    buffers.append((rows, rows[:, :, :2], rows[:, :, 2:]))
    pairs = torch.full((3, 5, 2, 2, 64), 7.0, device=device).half()
    buffers.append((pairs, pairs[:, :, :, 0], pairs[:, :, :, 1]))
    heads = torch.full((2, 3, 2, 5, 64), 7.0, device=device).half()
    buffers.append((heads, heads[0].permute(0, 2, 1, 3), heads[1].permute(0, 2, 1, 3)))
    tokens = torch.full((5, 3, 2, 2, 64), 7.0, device=device).half()
    buffers.append((tokens, tokens[:, :, 0].transpose(0, 1), tokens[:, :, 1].transpose(0, 1)))
    for whole, k, v in buffers:
        backend.kv_read_int4(cache, k, v, starts)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
        assert not torch.any(whole == 7)
