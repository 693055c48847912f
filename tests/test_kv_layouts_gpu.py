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


def test_attention_beside_its_queries(backend, device):
    """Outputs among the queries' rows, head by head, and heads as the slowest axis; queries of stride 0."""
    cache, g = _held(backend, device, 3, 2, 64, 64)
    n = torch.tensor([64, 5, 40], device=device, dtype=torch.int32)
    q = torch.randn((3, 4, 64), generator=g, device=device).half()
    want = backend.gqa_attention_int4(q, cache, torch.empty_like(q), n)
    for shape, parts in (((3, 4, 2, 64), lambda b: (b[:, :, 0], b[:, :, 1])), ((3, 2, 4, 64), lambda b: (b[:, 0], b[:, 1])),
                         ((4, 2, 3, 64), lambda b: (b[:, 0].transpose(0, 1), b[:, 1].transpose(0, 1)))):
        a, out = parts(torch.zeros(shape, device=device).half())
        a.copy_(q)
        backend.gqa_attention_int4(a, cache, out, n)
        assert torch.equal(out, want) and torch.equal(a, q)
    one = q[:1].expand(3, 4, 64)
    out = backend.gqa_attention_int4(one, cache, torch.empty_like(q), n)
    assert torch.equal(out, backend.gqa_attention_int4(one.contiguous(), cache, torch.empty_like(q), n))
    with pytest.raises(ValueError, match="share"):
        backend.gqa_attention_int4(q, cache, torch.empty((1, 4, 64), device=device).half().expand(3, 4, 64), n)
