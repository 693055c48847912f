"""Selecting pages by their bounds: the pages of the restatement exactly, ties, forced pages, odd scores.

Scores are float32 roundings of sums in float64 whose products are exact, so two orders of adding agree but for
a sum within 2^-50 of itself of a rounding border; inputs here are 16-bit values of like size."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.paged_ref import np64, scattered, scores, select
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _make(device, seed, needs, page, kvh, dim, dt):
    g = torch.Generator(device=device).manual_seed(seed)
    pages = sum(needs) + 3
    cache = PagedKvCache.allocate(pages, kvh, page, dim, dt, bounds=True, device=device)
    a, b = (torch.randn((pages, kvh, dim), generator=g, device=device) * 1.5 for _ in range(2))
    cache.k_bounds.copy_(torch.stack((torch.minimum(a, b), torch.maximum(a, b)), 2))
    return cache, scattered(np.random.default_rng(seed), needs, pages), g


def _check(backend, device, cache, table, lengths, q, count, first, last, limit=None):
    rows, kvh = len(lengths), cache.kv_heads
    got = torch.full((rows, kvh, count), -5, device=device, dtype=torch.int32)
    back = backend.select_pages(q, cache, torch.tensor(table, device=device), torch.tensor(lengths, device=device, dtype=torch.int32), got,
                                first_pages=first, last_pages=last, max_length=limit)
    assert back is got
    b = np64(cache.k_bounds)
    for r, n in enumerate(lengths):
        n = max(0, min(n, table.shape[1] * cache.page_size, limit or 1 << 30))
        pages = -(-n // cache.page_size)
        s = scores(np64(q[r]), b, table[r], pages)
        for j in range(kvh):
            assert got[r, j].tolist() == select(s[j], count, first, last), (r, j)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,dim,page", [(8, 2, 64, 16), (10, 2, 128, 64), (4, 4, 256, 32), (16, 1, 64, 256), (40, 1, 128, 16)])
def test_selection(backend, device, dtype, heads, kvh, dim, page):
    needs = [0, 1, 5, 63, 64, 65, 300]
    lengths = [0, 1, 5 * page - 3, 63 * page, 64 * page - 1, 64 * page + 1, 300 * page - 2]
    cache, table, g = _make(device, dim + page, needs, page, kvh, dim, _DT[dtype])
    q = torch.randn((len(needs), heads, dim), generator=g, device=device).to(_DT[dtype])
    for count, first, last in ((1, 0, 0), (5, 1, 2), (64, 0, 1), (65, 2, 0), (400, 1, 1), (7, 3, 4)):
        _check(backend, device, cache, table, lengths, q, count, first, last)
    _check(backend, device, cache, table, lengths, q, 6, 1, 1, limit=40 * page + 7)


@pytest.mark.parametrize("pages,count", [(3000, 100), (5000, 4096), (1025, 1024), (2048, 1)])
def test_many_pages(backend, device, pages, count):
    cache, table, g = _make(device, pages, [pages, 17], 16, 1, 64, torch.float16)
    q = torch.randn((2, 4, 64), generator=g, device=device).half()
    _check(backend, device, cache, table, [pages * 16, 17 * 16], q, count, min(1, count - 1), 0)


def test_ties(backend, device):
    """Few distinct scores: the lower page of equal ones; a query of 0, for which all are equal (and +0 is -0)."""
    cache, table, g = _make(device, 1, [700, 700], 16, 2, 64, torch.bfloat16)
    kinds = torch.randint(0, 3, (cache.pages,), generator=g, device=device)
    cache.k_bounds.copy_(cache.k_bounds[:3].clone()[kinds])
    q = torch.randn((2, 4, 64), generator=g, device=device).bfloat16()
    for count in (1, 50, 300, 699):
        _check(backend, device, cache, table, [11200, 11190], q, count, 0, 1)
    zero = torch.zeros_like(q)
    zero[1] = -0.0
    _check(backend, device, cache, table, [11200, 11190], zero, 33, 1, 2)


def test_odd_scores(backend, device):
    """Infinite and NaN bounds, entries of the table that are no pages, the largest values."""
    cache, table, g = _make(device, 2, [100, 100, 100], 32, 1, 64, torch.float16)
    q = torch.randn((3, 4, 64), generator=g, device=device).half()
    cache.k_bounds[int(table[0, 30]), 0, 1, 5] = float("inf")
    cache.k_bounds[int(table[0, 60]), 0, 0, 9] = float("nan")
    cache.k_bounds[int(table[0, 70]), 0, 0, 11] = float("-inf")
    cache.k_bounds[int(table[0, 80]), 0, 1, 12] = 65504.0
    table[1, 50], table[1, 99], table[1, 20] = -3, cache.pages, 1 << 30
    for count in (2, 3, 4, 6, 20):
        _check(backend, device, cache, table, [3200, 3200, 3199], q, count, 1, 0)


def test_strided_queries(backend, device):
    cache, table, g = _make(device, 3, [40, 40], 16, 2, 128, torch.float16)
    rows = torch.randn((2, 5 + 8 * 128), generator=g, device=device).half()
    q = rows[:, 5:5 + 4 * 128].view(2, 4, 128)
    a = _check(backend, device, cache, table, [640, 600], q, 9, 1, 2)
    wide = PagedKvCache(cache.k_pages, cache.v_pages, torch.cat((cache.k_bounds, cache.k_bounds), 1)[:, :2])
    assert torch.equal(a, _check(backend, device, wide, table, [640, 600], q, 9, 1, 2))
