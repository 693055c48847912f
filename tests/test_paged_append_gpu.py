"""Appending to the paged cache with the rotation on the way: rotated values have the bits of
``rotary_rows`` and lie within its bound of float64, every token is where its table says, bounds are the
extremes of the keys as they are stored, and nothing else changes.

Rotation: the angle is formed in binary64 and reduced there; in turns it is rounded to binary32 once
(2^-25 of half a turn) and doubled, sine and cosine are good to 2^-22, so a turned value is off by at most
2 pi 2^-25 + 2^-22 + 3 roundings of 2^-24 of (|a| + |b|) amplitude, below 2^-20 of it, and half a step of its type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref
from tests.paged_ref import np64, places, row_counts, same_bits, scattered
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _junk(cache, seed):
    """Every bit pattern."""
    g = torch.Generator(device=cache.device).manual_seed(seed)
    for t in (cache.k_pages, cache.v_pages, cache.k_bounds):
        if t is not None:
            t.copy_(torch.randint(-(2 ** 15), 2 ** 15, t.shape, generator=g, device=t.device, dtype=torch.int16).view(t.dtype))


def _copy(cache):
    return PagedKvCache(cache.k_pages.clone(), cache.v_pages.clone(), None if cache.k_bounds is None else cache.k_bounds.clone())


def _check(backend, cache, before, q, k, v, q_out, table, starts, cu, inv_freq, interleaved=False, amplitude=1.0, q_before=None):
    tokens, rows = k.shape[0], len(starts)
    counts = row_counts(cu, rows, tokens)
    firsts = cu[:-1] if cu is not None else [r * (tokens // rows) for r in range(rows)]
    pos = torch.zeros(tokens, dtype=torch.int64)
    used = torch.zeros(tokens, dtype=torch.bool)
    for r in range(rows):
        for i in range(counts[r]):
            pos[firsts[r] + i], used[firsts[r] + i] = starts[r] + i, True
    kt, qt = k.clone(), None if q is None else q.clone()
    if inv_freq is not None:
        backend.rotary_rows(q if q is not None else k, k if q is not None else None, pos.to(k.device), inv_freq,
                            qt if q is not None else kt, kt if q is not None else None, interleaved=interleaved, amplitude=amplitude)
    if q is not None:
        assert same_bits(q_out[used], qt[used])
        if q_before is not None:
            assert same_bits(q_out[~used], q_before[~used])
    want_k, want_v = before.k_pages.clone(), before.v_pages.clone()
    want_b = None if before.k_bounds is None else before.k_bounds.clone()
    for r in range(rows):
        runs = {}
        for i, (page, slot) in enumerate(places(table[r], starts[r], counts[r], cache.page_size)):
            if 0 <= page < cache.pages:
                want_k[page, :, slot], want_v[page, :, slot] = kt[firsts[r] + i], v[firsts[r] + i]
                runs.setdefault(page, []).append(slot)
        for page, slots in runs.items() if want_b is not None else ():
            keys = want_k[page][:, slots].float()
            lo, hi = keys.amin(1), keys.amax(1)
            if slots[0] != 0:
                lo, hi = torch.minimum(want_b[page, :, 0].float(), lo), torch.maximum(want_b[page, :, 1].float(), hi)
            want_b[page, :, 0], want_b[page, :, 1] = lo.to(cache.dtype), hi.to(cache.dtype)
    assert same_bits(cache.k_pages, want_k) and same_bits(cache.v_pages, want_v)
    if want_b is not None:
        got, nan = cache.k_bounds, torch.isnan(want_b)
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want_b[~nan])


def _inv_freq(r, device):
    return 500000.0 ** (-torch.arange(0, r, 2, device=device, dtype=torch.float64) / r)


def _operands(device, seed, tokens, heads, kv_heads, dim, dt):
    g = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn((tokens, h, dim), generator=g, device=device) * 2).to(dt) for h in (heads, kv_heads, kv_heads)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,page,rotary,interleaved", [(64, 16, 64, False), (64, 32, 16, True), (128, 64, 64, True), (128, 16, 128, False),
                                                         (256, 128, 128, False), (256, 256, 256, True), (128, 32, 34, False), (64, 16, 6, True)])
@pytest.mark.parametrize("bounds", [False, True])
def test_ragged_rows(backend, device, dtype, dim, page, rotary, interleaved, bounds):
    """Rows of none, one and many tokens, that begin and end inside pages, a row outside the table, bad entries."""
    rng = np.random.default_rng(dim + page)
    counts, starts = [1, 0, 2 * page + 5, 17, page, 1, 3, 5], [3, 4, page - 2, 0, page, 4 * page - 1, -2, 4 * page - 3]
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    cache = PagedKvCache.allocate(40, 3, page, dim, _DT[dtype], bounds=bounds, device=device)
    _junk(cache, page)
    before = _copy(cache)
    table = scattered(rng, [4] * 8, 40)
    table[3, 0], table[4, 1] = -7, 40                          # no pages
    tokens = cu[-1] + 4                                        # four tokens behind the last row
    q, k, v = _operands(device, dim, tokens, 6, 3, dim, _DT[dtype])
    out = torch.full_like(q, 7.0)
    f = _inv_freq(rotary, device)
    backend.rotary_append_paged(cache, q, k, v, torch.from_numpy(table).to(device), torch.tensor(starts, device=device, dtype=torch.int32), f,
                                out, cu_tokens=torch.tensor(cu, device=device, dtype=torch.int32), interleaved=interleaved, amplitude=1.25)
    _check(backend, cache, before, q, k, v, out, table, starts, cu, f, interleaved, 1.25, torch.full_like(q, 7.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_against_float64(backend, device, dtype):
    dt, dim, starts = _DT[dtype], 128, [0, 1000003, 77]
    q, k, v = _operands(device, 3, 3 * 5, 8, 2, dim, dt)
    width = 1000192 // 256
    table = np.full((3, width), -1, dtype=np.int32)
    for r, s in enumerate(starts):
        table[r, s // 256] = r
    cache = PagedKvCache.allocate(3, 2, 256, dim, dt, device=device)
    f = _inv_freq(dim, device)
    out = backend.rotary_append_paged(cache, q, k, v, torch.from_numpy(table).to(device), torch.tensor(starts, device=device, dtype=torch.int32), f,
                                      torch.empty_like(q), amplitude=1.3)
    pos = [s + i for s in starts for i in range(5)]
    stored = torch.stack([cache.k_pages[t // 5, :, p % 256] for t, p in enumerate(pos)])
    info = torch.finfo(dt)
    for got, x in ((out, q), (stored, k)):
        want = step_ref.rotary(np64(x), pos, f.cpu().numpy(), False, 1.3)
        mag = np.abs(np64(x))
        mag = 1.3 * np.concatenate([mag[..., :64] + mag[..., 64:]] * 2, -1)
        assert np.all(np.abs(np64(got) - want) <= mag * 2.0 ** -20 + info.eps / 2 * np.abs(want) * (1 + 2.0 ** -10) + info.tiny * info.eps)


@pytest.mark.parametrize("rows,heads,kv_heads,dim,page", [(1, 32, 8, 64, 16), (8, 40, 10, 128, 64), (64, 8, 1, 256, 128), (70, 2, 2, 64, 32)])
def test_a_token_a_row_in_place(backend, device, rows, heads, kv_heads, dim, page):
    """One token for every row, q in place, and the next ones after it: bounds follow page by page."""
    rng = np.random.default_rng(rows)
    cache = PagedKvCache.allocate(2 * rows + 3, kv_heads, page, dim, torch.bfloat16, bounds=True, device=device)
    _junk(cache, rows)
    cache.k_bounds.nan_to_num_(0.0, 3.0, -3.0)
    table = scattered(rng, [2] * rows, 2 * rows + 3)
    f = _inv_freq(dim, device)
    starts = [(page - 1 + 5 * r) % (2 * page - 3) for r in range(rows)]
    for step in range(3):
        before = _copy(cache)
        q, k, v = _operands(device, rows + step, rows, heads, kv_heads, dim, torch.bfloat16)
        q0 = q.clone()
        now = [s + step for s in starts]
        got = backend.rotary_append_paged(cache, q, k, v, torch.from_numpy(table).to(device), torch.tensor(now, device=device, dtype=torch.int32), f)
        assert got is q
        _check(backend, cache, before, q0, k, v, q, table, now, None, f)


def test_one_by_one_equals_at_once(backend, device):
    q, k, v = _operands(device, 5, 2 * 83, 4, 2, 64, torch.float16)
    k[40, 1, 7] = float("nan")
    k[90, 0, 3] = float("inf")
    a, b = (PagedKvCache.allocate(12, 2, 32, 64, bounds=True, device=device) for _ in range(2))
    table = torch.tensor([[5, 2, 9, 11], [0, 7, 3, 8]], device=device, dtype=torch.int32)
    f = _inv_freq(64, device)
    starts = torch.tensor([0, 32], device=device, dtype=torch.int32)
    out = backend.rotary_append_paged(a, q, k, v, table, starts, f, torch.empty_like(q))
    for i in range(83):
        pick = torch.tensor([i, 83 + i], device=device)
        one = backend.rotary_append_paged(b, q[pick], k[pick], v[pick], table, starts + i, f)
        assert same_bits(one, out[pick])
    assert same_bits(a.k_pages, b.k_pages) and same_bits(a.v_pages, b.v_pages)
    assert torch.equal(a.k_bounds.nan_to_num(1e4), b.k_bounds.nan_to_num(1e4)) and torch.isnan(a.k_bounds[2, 1, :, 7]).all()


@pytest.mark.parametrize("layout", ["heads first", "tokens first", "side by side", "a layer of many"])
def test_layouts_and_strides(backend, device, layout):
    """Caches as views, q, k and v as odd parts of a fused row, without a rotation and without q."""
    dt, pages, kvh, page, dim = torch.float16, 9, 2, 16, 64
    g = torch.Generator(device=device).manual_seed(3)
    if layout == "tokens first":
        k_store, v_store = (torch.randn((pages, page, kvh, dim), generator=g, device=device).to(dt) for _ in range(2))
        cache = PagedKvCache(k_store.transpose(1, 2), v_store.transpose(1, 2))
    elif layout == "side by side":
        store = torch.randn((pages, page, 2, kvh, dim), generator=g, device=device).to(dt)
        cache = PagedKvCache(store[:, :, 0].transpose(1, 2), store[:, :, 1].transpose(1, 2))
    elif layout == "a layer of many":
        store = torch.randn((pages, 3, 2, kvh, page, dim), generator=g, device=device).to(dt)
        cache = PagedKvCache(store[:, 1, 0], store[:, 1, 1])
    else:
        cache = PagedKvCache(*(torch.randn((pages, kvh, page, dim), generator=g, device=device).to(dt) for _ in range(2)))
    before = _copy(cache)
    whole = None if layout in ("heads first", "tokens first") else store.clone()
    qkv = torch.randn((22, 1 + 8 * dim), generator=g, device=device).to(dt)
    q, k, v = qkv[:, 1:1 + 4 * dim].view(22, 4, dim), qkv[:, 1 + 4 * dim:1 + 6 * dim].view(22, 2, dim), qkv[:, 1 + 6 * dim:].view(22, 2, dim)
    table = scattered(np.random.default_rng(2), [3, 3], pages)
    starts, f = [5, 30], _inv_freq(dim, device)
    args = (torch.from_numpy(table).to(device), torch.tensor(starts, device=device, dtype=torch.int32))
    wide = torch.full((22, 4, dim + 3), 5.0, device=device, dtype=dt)
    out = wide[:, :, 1:dim + 1]
    backend.rotary_append_paged(cache, q, k, v, *args, f, out)
    _check(backend, cache, before, q, k, v, out, table, starts, None, f)
    assert torch.all(wide[..., 0] == 5.0) and torch.all(wide[..., dim + 1:] == 5.0)
    before = _copy(cache)
    assert backend.rotary_append_paged(cache, None, v, k, *args, None) is None           # neither q nor a rotation
    _check(backend, cache, before, None, v, k, None, table, starts, None, None)
    before = _copy(cache)
    backend.rotary_append_paged(cache, None, k, v, *args, f)
    _check(backend, cache, before, None, k, v, None, table, starts, None, f)
    if layout == "a layer of many":
        assert same_bits(store[:, 0], whole[:, 0]) and same_bits(store[:, 2], whole[:, 2])


def test_far_pages_and_wild_counts(backend, device):
    """Places past 2^31 elements, and cu_tokens that no program should give: nothing outside the operands is touched."""
    page, kvh, dim = 256, 8, 256
    pages = (1 << 31) // (page * kvh * dim) + 3
    cache = PagedKvCache.allocate(pages, kvh, page, dim, device=device)
    q, k, v = _operands(device, 8, 3, 8, kvh, dim, torch.float16)
    table = torch.tensor([[pages - 1, pages - 2]], device=device, dtype=torch.int32)
    backend.rotary_append_paged(cache, q, k, v, table, torch.tensor([page - 1], device=device, dtype=torch.int32), None)
    assert same_bits(cache.k_pages[pages - 1, :, page - 1], k[0]) and same_bits(cache.v_pages[pages - 2, :, 1], v[2])
    small = PagedKvCache.allocate(4, 2, 16, 64, device=device)
    q, k, v = _operands(device, 8, 9, 2, 2, 64, torch.float16)
    table = torch.tensor([[0, 1], [2, 3]], device=device, dtype=torch.int32)
    for cu in ([-5, 3, 900], [9, 2, 9], [0, 0, 0], [4, 4, 2]):
        out = torch.full((11, 2, 64), 9.0, device=device, dtype=torch.float16)
        backend.rotary_append_paged(small, q, k, v, table, torch.zeros(2, device=device, dtype=torch.int32), None, out[1:10],
                                    cu_tokens=torch.tensor(cu, device=device, dtype=torch.int32))
        assert torch.all(out[0] == 9.0) and torch.all(out[10] == 9.0)
