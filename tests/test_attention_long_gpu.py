"""Attention over long rows of the 4-bit cache within bounds that reject a lost or repeated tile: by the
depth of the kernel's additions, and exactly, with equal weights and values that mark every token."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import attention_bound, step_ref
from thintensor_amd.kv_cache import Int4KvCache

pytestmark = pytest.mark.gpu


def _shared(cache, rows):
    return Int4KvCache(*[t.expand(rows, *t.shape[1:]) for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)])


def _lengths(rows, capacity):
    some = [capacity, 0, 1, 8192, 8193, 16385, 32, 4096, 24577, capacity - 1, 8160, 33]
    return [min(some[b], capacity) if b < len(some) else (37 * b) % capacity for b in range(rows)]


@pytest.mark.parametrize("dim,rows,kv_heads,heads,window,first,max_length", [
    (64, 64, 8, 24, 0, 0, None), (128, 64, 8, 8, 0, 0, None), (256, 70, 4, 16, 0, 0, None), (128, 33, 1, 48, 0, 0, None),
    (128, 3, 2, 10, 0, 0, None), (64, 1, 1, 8, 0, 0, None), (256, 2, 2, 2, 0, 0, None), (64, 9, 2, 34, 0, 0, None),
    (128, 64, 8, 16, 20000, 33, None), (64, 4, 2, 8, 30001, 4, None), (128, 64, 8, 8, 8200, 0, None), (128, 64, 8, 8, 0, 0, 8192),
    (64, 64, 8, 8, 0, 0, 20001), (64, 5, 1, 1, 2, 25000, None)])
def test_every_token_counts_once(backend, device, dim, rows, kv_heads, heads, window, first, max_length):
    """Weights are equal (a scale of 0); the tokens behind a row's length mark dims as well."""
    capacity = 36000
    at = attention_bound.marks(capacity, kv_heads, dim, dim + rows)
    g = torch.Generator(device=device).manual_seed(rows)
    cache = Int4KvCache.allocate(1, kv_heads, capacity, dim, 32, device)
    k = torch.randn((1, capacity, kv_heads, dim), generator=g, device=device).half()
    v = torch.zeros((1, capacity, kv_heads, dim), device=device).half()
    v.scatter_(3, torch.from_numpy(at).to(device)[None, :, :, None], 15.0)
    backend.kv_append_int4(cache, k, v, torch.zeros(1, device=device, dtype=torch.int32))
    lengths = _lengths(rows, capacity)
    q = torch.randn((rows, heads, dim), generator=g, device=device).half()
    out = torch.full_like(q, 5.0)
    backend.gqa_attention_int4(q, _shared(cache, rows), out, torch.tensor(lengths, device=device, dtype=torch.int32), scale=0.0,
                               window=window, first_tokens=first, max_length=max_length)
    got = out.double().cpu().numpy()
    for b, n in enumerate(lengths):
        n = min(n, max_length or capacity)
        t = np.arange(n)
        if window:
            t = t[(t >= n - window) | (t < first)]
        want = np.repeat(attention_bound.marked(at, dim, t), heads // kv_heads, 0)
        err = np.abs(got[b] - want)
        assert np.all(err <= attention_bound.marked_bound(want, torch.finfo(q.dtype))), (b, n, float(err.max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,rows,kv_heads,heads,capacity", [
    (64, 64, 8, 8, 36000), (128, 64, 8, 8, 36000), (128, 2, 1, 16, 36000), (256, 66, 4, 4, 20000), (128, 1, 1, 4, 131072),
    (64, 3, 2, 8, 20000)])
def test_long_rows(backend, device, dtype, dim, rows, kv_heads, heads, capacity):
    """Scores of about one, so that every tile weighs; the same rows in another order give the same bits."""
    g = torch.Generator(device=device).manual_seed(dim + rows + capacity)
    cache = Int4KvCache.allocate(1, kv_heads, capacity, dim, 64, device)
    k = torch.randn((1, capacity, kv_heads, dim), generator=g, device=device)
    k += torch.randn((1, 1, kv_heads, dim), generator=g, device=device) * 1.5
    backend.kv_append_int4(cache, k, torch.randn((1, capacity, kv_heads, dim), generator=g, device=device),
                           torch.zeros(1, device=device, dtype=torch.int32))
    held = []
    for codes, (s, m) in (
            (step_ref.unpack_k(cache.k_codes[0].cpu().numpy()), np.moveaxis(cache.k_scales[0].double().cpu().numpy(), -1, 0)),
            (step_ref.unpack_v(cache.v_codes[0].cpu().numpy()), step_ref.unpack_v_scales(cache.v_scales[0].double().cpu().numpy()))):
        held.append(step_ref.dequantize(codes, s, m))
    lengths = _lengths(rows, capacity)
    q = torch.randn((rows, heads, dim), generator=g, device=device).to(dtype)
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    out, scale = torch.full_like(q, 5.0), dim ** -0.5 / 16
    backend.gqa_attention_int4(q, _shared(cache, rows), out, n, scale=scale)
    tiles, parts = attention_bound.tiles_per_wave(rows * kv_heads * -(-heads // kv_heads // 16), capacity)
    for b in [x for x in (0, 4, 5, 7, 8) if x < rows]:
        want, mag, reach, peak = attention_bound.attention(q[b].double().cpu().numpy(), held[0][:, :lengths[b]], held[1][:, :lengths[b]],
                                                           float(np.float32(scale)))
        err = np.abs(out[b].double().cpu().numpy() - want)
        limit = attention_bound.bound(want, mag, reach, peak, lengths[b], tiles, parts, torch.finfo(dtype))
        assert np.all(err <= limit), (b, lengths[b], float((err - limit).max()), float(err.max()))
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rows)).to(device)
    mixed = torch.empty_like(q)
    backend.gqa_attention_int4(q[order].contiguous(), _shared(cache, rows), mixed, n[order].contiguous(), scale=scale)
    assert torch.equal(mixed, out[order])


@pytest.mark.parametrize("scale", [1e38, 3e38])
@pytest.mark.parametrize("tokens", [50, 4000])
def test_scores_past_binary32(backend, device, scale, tokens):
    """A score past the largest value makes its head NaN, scores all past the smallest one do without a
    sink; a head of scores 0 is the mean of V where the scale itself is in range, whatever the others are."""
    cache = Int4KvCache.allocate(1, 1, tokens + 32, 64, 32, device)
    g = torch.Generator(device=device).manual_seed(tokens)
    k = torch.rand((1, tokens, 1, 64), generator=g, device=device) + 1
    v = torch.randn((1, tokens, 1, 64), generator=g, device=device)
    backend.kv_append_int4(cache, k, v, torch.zeros(1, device=device, dtype=torch.int32))
    q = torch.ones((1, 3, 64), device=device).half()
    q[0, 1] = -1.0
    q[0, 2] = 0.0
    n = torch.tensor([tokens], device=device, dtype=torch.int32)
    out = backend.gqa_attention_int4(q, cache, torch.empty_like(q), n, scale=scale)
    sinks = torch.zeros(3, device=device)
    beside = backend.gqa_attention_int4(q, cache, torch.empty_like(q), n, scale=scale, sinks=sinks)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(beside[0, 0]).all()
    if scale < 2e38:
        assert torch.count_nonzero(beside[0, 1]) == 0
        mean = backend.kv_read_int4(cache, torch.empty_like(k), torch.empty_like(v), torch.zeros(1, device=device, dtype=torch.int32))[1]
        mean = mean.double().sum((0, 1, 2))
        assert torch.all((out[0, 2].double() - mean / tokens).abs() <= 2.0 ** -10 * (mean / tokens).abs() + 2.0 ** -18)
        assert torch.all((beside[0, 2].double() - mean / (tokens + 1)).abs() <= 2.0 ** -10 * (mean / (tokens + 1)).abs() + 2.0 ** -18)
