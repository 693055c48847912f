"""Attention over a paged cache, behind shared pages and over selected pages, against float64 within the
bound that ``tests/paged_ref.py`` derives, and exactly where equal weights meet values that mark every token."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.paged_ref import attention, attention_bound, np64, row_counts, same_bits, scattered
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _make(device, seed, lengths, page, kv_heads, dim, dtype, shared=0, spare=3):
    """A cache with keys of uneven channel means in scattered pages, junk of every bit pattern (NaN among it) in
    all slots that no row's length reaches, and the table, -1 where no token needs an entry."""
    g = torch.Generator(device=device).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = _DT[dtype]
    needs = [-(-n // page) for n in lengths]
    pages = shared + sum(max(0, n - shared) for n in needs) + spare
    table = scattered(rng, needs, pages, shared)
    cache = PagedKvCache.allocate(pages, kv_heads, page, dim, dt, bounds=True, device=device)
    for t in (cache.k_pages, cache.v_pages):
        t.copy_(torch.randint(-(2 ** 15), 2 ** 15, t.shape, generator=g, device=device, dtype=torch.int16).view(dt))
        t.masked_fill_(torch.rand(t.shape, generator=g, device=device) < 0.2, float("nan"))
    means = torch.randn((kv_heads, 1, dim), generator=g, device=device) * 1.5
    filled = {}
    for r, n in enumerate(lengths):
        for p in range(needs[r]):
            filled[int(table[r, p])] = max(filled.get(int(table[r, p]), 0), min(page, n - p * page))
    for i, m in filled.items():
        cache.k_pages[i, :, :m] = (torch.randn((kv_heads, m, dim), generator=g, device=device) + means).to(dt)
        cache.v_pages[i, :, :m] = torch.randn((kv_heads, m, dim), generator=g, device=device).to(dt)
    return cache, table, g


def _i32(x, device):
    return torch.tensor(np.asarray(x), device=device, dtype=torch.int32)


def _run(backend, device, cache, table, lengths, q, cu=None, **kw):
    out = torch.full_like(q, 9.0)
    sel = kw.pop("selected", None)
    got = backend.gqa_attention_paged(q, cache, _i32(table, device), _i32(lengths, device), out,
                                      cu_tokens=None if cu is None else _i32(cu, device),
                                      selected=None if sel is None else _i32(sel, device), **kw)
    assert got is out
    return out


def _check(cache, table, lengths, q, out, cu=None, **kw):
    kw.pop("shared_pages", None)
    counts = row_counts(cu, len(lengths), q.shape[0])
    first, used = (cu[0], cu[-1]) if cu is not None else (0, q.shape[0])
    if kw.get("sinks") is not None:
        kw["sinks"] = np64(kw["sinks"])
    want, mag, reach, seen, peak = attention(np64(q[first:used]), np64(cache.k_pages), np64(cache.v_pages), table, lengths, counts, cache.page_size, **kw)
    got = np64(out[first:used])
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    with np.errstate(invalid="ignore"):
        off = np.where(fine, np.abs(got - want) - attention_bound(want, mag, reach, seen, peak, q.dtype), 0.0)
    assert np.nanmax(off, initial=0.0) <= 0 and not np.isnan(off).any(), (np.unravel_index(off.argmax(), off.shape), float(off.max()))
    assert torch.all(out[used:] == 9.0) and torch.all(out[:first] == 9.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens(backend, device, dtype, dim, page):
    """Lengths of none, one, around pages and tiles; rows with nothing."""
    lengths = [0, 1, 15, 16, 17, 31, 33, page, page + 1, 3 * page - 1, 300]
    cache, table, g = _make(device, dim + page, lengths, page, 2, dim, dtype)
    q = torch.randn((len(lengths), 10, dim), generator=g, device=device).to(_DT[dtype])
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 10), (16, 1), (17, 1), (64, 2), (3, 1)])
def test_head_layouts(backend, device, dtype, heads, kv_heads):
    lengths = [130, 0, 700, 1]
    cache, table, g = _make(device, heads, lengths, 32, kv_heads, 64, dtype)
    q = torch.randn((4, heads, 64), generator=g, device=device).to(_DT[dtype])
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(2, 8, 2, 64), (4, 8, 2, 128), (3, 5, 1, 128), (7, 4, 2, 256), (33, 8, 2, 64), (70, 2, 2, 128)])
def test_several_tokens(backend, device, dtype, tokens, heads, kv_heads, dim):
    """As many queries for every row; rows shorter than their queries leave some that see nothing."""
    lengths = [tokens, tokens + 1, 200, 1, 0, 391]
    cache, table, g = _make(device, tokens, lengths, 16, kv_heads, dim, dtype)
    q = torch.randn((len(lengths) * tokens, heads, dim), generator=g, device=device).to(_DT[dtype])
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q))


_RAGGED = [1, 0, 150, 17, 1, 64, 3], [40, 33, 150, 300, 1, 70, 0]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window", [(8, 2, 64, 16, 0), (8, 2, 128, 64, 0), (5, 1, 256, 32, 0), (4, 4, 128, 256, 40), (16, 1, 64, 64, 1),
                                                            (10, 2, 128, 16, 130)])
@pytest.mark.parametrize("sinks", [False, True])
def test_ragged_chunks(backend, device, dtype, heads, kv_heads, dim, page, window, sinks):
    counts, lengths = _RAGGED
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    cache, table, g = _make(device, heads + dim, lengths, page, kv_heads, dim, dtype)
    q = torch.randn((cu[-1] + 5, heads, dim), generator=g, device=device).to(_DT[dtype])
    kw = dict(window=window, sinks=torch.randn(heads, generator=g, device=device) * 2 if sinks else None)
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, cu, **kw), cu, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window", [1, 16, 33, 128, 5000])
def test_windows_and_sinks(backend, device, dtype, window):
    lengths = [900, 1, 0, 127, 128, 129, 480]
    cache, table, g = _make(device, window, lengths, 16, 2, 64, dtype)
    q = torch.randn((len(lengths), 8, 64), generator=g, device=device).to(_DT[dtype])
    for sinks in (None, torch.randn(8, generator=g, device=device).to(_DT[dtype]), torch.randn(8, generator=g, device=device) * 30):
        kw = dict(window=window, sinks=sinks)
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, **kw), **kw)


def test_long_rows_among_short_ones(backend, device):
    lengths = [9001, 1, 0, 2500, 63]
    cache, table, g = _make(device, 1, lengths, 64, 1, 128, "bf16")
    q = torch.randn((5, 8, 128), generator=g, device=device).bfloat16()
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q))
    for limit in (1, 64, 2499, 1 << 20):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, max_length=limit), max_length=limit)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,shared", [(6, 8, 2, 64, 16, 9), (3, 40, 10, 128, 64, 3), (40, 8, 1, 128, 32, 20), (2, 2, 1, 256, 16, 30),
                                                                 (70, 16, 2, 64, 64, 2), (1, 8, 2, 64, 16, 9)])
def test_shared_pages(backend, device, dtype, rows, heads, kv_heads, dim, page, shared):
    """Rows that end behind, at the end of, and inside the shared pages, and one with nothing."""
    base = shared * page
    lengths = [base + 1, base, base - page - 3, 0, base + 77, 1, base + 3 * page, base - 1] * 9
    lengths = lengths[:rows]
    if rows == 1:
        lengths = [base + 20]
    cache, table, g = _make(device, rows + dim, lengths, page, kv_heads, dim, dtype, shared)
    # the junk behind a shorter row's end is what longer rows read: fill the shared pages for all
    for p in table[0, :shared]:
        cache.k_pages[p] = torch.randn(cache.k_pages[p].shape, generator=g, device=device).to(cache.dtype)
        cache.v_pages[p] = torch.randn(cache.v_pages[p].shape, generator=g, device=device).to(cache.dtype)
    for tokens in (1, 3):
        q = torch.randn((rows * tokens, heads, dim), generator=g, device=device).to(_DT[dtype])
        for kw in (dict(shared_pages=shared), dict(shared_pages=shared, window=base // 2 + 5),
                   dict(shared_pages=shared - 1, sinks=torch.randn(heads, generator=g, device=device))):
            _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, **kw), **kw)


def test_shared_pages_ragged(backend, device):
    counts, lengths = [5, 0, 90, 1, 1, 33], [150, 200, 260, 64, 10, 129]
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    cache, table, g = _make(device, 4, lengths, 16, 2, 128, "bf16", 8)
    for p in table[0, :8]:
        cache.k_pages[p].normal_(generator=g)
        cache.v_pages[p].normal_(generator=g)
    q = torch.randn((cu[-1] + 2, 10, 128), generator=g, device=device).bfloat16()
    out = _run(backend, device, cache, table, lengths, q, cu, shared_pages=8)
    _check(cache, table, lengths, q, out, cu)
    # only row 0's entries of the shared pages are read
    other = table.copy()
    other[1:, :8] = -1
    assert same_bits(out, _run(backend, device, cache, other, lengths, q, cu, shared_pages=8))


def test_all_pages_shared(backend, device):
    lengths = [160] * 20
    cache, table, g = _make(device, 4, lengths, 16, 2, 64, "f16", 10)
    q = torch.randn((20, 8, 64), generator=g, device=device).half()
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, shared_pages=10))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,page,count", [(64, 16, 5), (128, 32, 3), (64, 64, 40), (256, 16, 1), (128, 256, 2), (64, 128, 7)])
def test_selected_pages(backend, device, dtype, dim, page, count):
    rng = np.random.default_rng(count)
    lengths = [20 * page - 5, 0, 3, 7 * page, 11 * page + 1]
    cache, table, g = _make(device, page, lengths, page, 3, dim, dtype)
    sel = -np.ones((5, 3, count), dtype=np.int32)
    for r, n in enumerate(lengths):
        for j in range(3):
            held = rng.permutation(max(1, -(-n // page)) + 2)[:count]          # some past the row's end
            sel[r, j, :len(held)] = held
    sel[3, 1] = -1                                                             # nothing at all
    q = torch.randn((5, 6, dim), generator=g, device=device).to(_DT[dtype])
    for kw in (dict(), dict(sinks=torch.randn(6, generator=g, device=device)), dict(window=2 * page + 3)):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, selected=sel, **kw), selected=sel, **kw)


def test_all_pages_selected_equals_dense(backend, device):
    lengths = [500, 333]
    cache, table, g = _make(device, 8, lengths, 32, 2, 128, "f16")
    q = torch.randn((2, 8, 128), generator=g, device=device).half()
    sel = np.tile(np.arange(16, dtype=np.int32), (2, 2, 1))
    out = _run(backend, device, cache, table, lengths, q, selected=sel)
    _check(cache, table, lengths, q, out)
    back = _run(backend, device, cache, table, lengths, q, selected=sel[..., ::-1].copy())   # any order
    _check(cache, table, lengths, q, back)


@pytest.mark.parametrize("tokens", [1, 40])
def test_bad_table_entries(backend, device, tokens):
    """Entries that are no pages: NaN for the queries that need them, none for the others."""
    lengths = [100, 100, 100, 40]
    cache, table, g = _make(device, 5, lengths, 16, 2, 64, "f16")
    q = torch.randn((4 * tokens, 8, 64), generator=g, device=device).half()
    table[0, 1], table[1, 6], table[2, 0] = -1, cache.pages, 1 << 30
    for kw in (dict(), dict(window=30)):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, **kw), **kw)
    if tokens == 1:
        sel = np.tile(np.array([0, 2, 3], dtype=np.int32), (4, 2, 1))
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, selected=sel), selected=sel)
    table[0, 0] = -9                                          # row 0's entry, which every row reads
    out = _run(backend, device, cache, table, [20, 100, 16, 40], q, shared_pages=1)
    assert torch.isnan(out.view(4, tokens, -1)[:, -1]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [1, 24, 130])
def test_nan_and_infinities_out_of_sight(backend, device, dtype, tokens):
    """What a query may not see changes nothing: values and keys of later tokens that are not finite."""
    lengths = [tokens + 50, tokens]
    cache, table, g = _make(device, 6, lengths, 16, 2, 64, dtype)
    q = torch.randn((2 * tokens, 4, 64), generator=g, device=device).to(_DT[dtype])
    clean = _run(backend, device, cache, table, lengths, q, window=30)
    at = tokens // 2 + 50                                     # of row 0: seen by the later half of its queries
    page, slot = int(table[0, at // 16]), at % 16
    cache.v_pages[page, :, slot, 3] = float("nan")
    cache.v_pages[page, :, slot, 40] = float("inf")
    cache.k_pages[int(table[0, (at + 1) // 16]), 0, (at + 1) % 16, 5] = float("nan")
    out = _run(backend, device, cache, table, lengths, q, window=30)
    _check(cache, table, lengths, q, out, window=30)
    before = max(0, at - 50)                                  # the queries of row 0 that do not see it yet
    if tokens > 1:
        assert same_bits(out[:before], clean[:before]) and same_bits(out[tokens:], clean[tokens:])


def test_extreme_scores(backend, device):
    """Scores in the tens of thousands, equal ones, a scale of 0, negative ones; queries of 0."""
    lengths = [64, 65, 200]
    cache, table, g = _make(device, 7, lengths, 32, 1, 64, "bf16")
    q = torch.randn((3, 4, 64), generator=g, device=device).bfloat16()
    for scale in (0.0, -0.125, 3.0):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, scale=scale), scale=scale)
    _check(cache, table, lengths, q * 0, _run(backend, device, cache, table, lengths, q * 0))
    # one token takes everything: the others' weights are 0 exactly
    cache.k_pages[int(table[2, 1]), 0, 5] = 300.0
    big = torch.full_like(q, 300.0)
    out = _run(backend, device, cache, table, lengths, big)
    assert same_bits(out[2, 0], cache.v_pages[int(table[2, 1]), 0, 5])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,shared", [(1, 0), (1, 7), (5, 0), (64, 0), (150, 4)])
def test_every_token_counts_once(backend, device, dim, tokens, shared):
    """Equal weights, and values of a power of two that mark a token: for a query that sees n tokens, the output's
    dim d is the number of tokens t with t % dim == d over n.  Counts of at most 2^8 and their sums are exact in
    bf16 products; the quotient is rounded in binary32 and to bf16, 2^-8 + 2^-22 of it."""
    page, length = 16, 700
    lengths = [length, length - 13, tokens]
    needs = [-(-n // page) for n in lengths]
    pages = sum(needs) + 2
    rng = np.random.default_rng(tokens)
    table = scattered(rng, needs, pages, shared)
    cache = PagedKvCache.allocate(pages, 2, page, dim, torch.bfloat16, device=device)
    cache.v_pages.fill_(float("nan"))
    for r, n in enumerate(lengths):
        for t in range(n):
            row = torch.zeros(dim, device=device)
            row[t % dim] = 1.0
            cache.v_pages[int(table[r, t // page]), :, t % page] = row.bfloat16()
    for p in table[0, :shared]:
        assert not torch.isnan(cache.v_pages[int(p)]).any()
    q = torch.zeros((3 * tokens, 6, dim), device=device, dtype=torch.bfloat16)
    out = np64(_run(backend, device, cache, table, lengths, q, shared_pages=shared))
    for r, n in enumerate(lengths):
        for i in range(tokens):
            hi = n - (tokens - 1 - i)
            want = np.bincount(np.arange(max(hi, 0)) % dim, minlength=dim) / max(hi, 1)
            assert np.all(np.abs(out[r * tokens + i] - want) <= want * (2.0 ** -8 + 2.0 ** -20)), (r, i)


@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_strided_operands_in_place(backend, device, tokens):
    """q as an odd part of a fused row, out in place and as a view, a cache with its tokens before its heads."""
    lengths = [150, 131]
    cache, table, g = _make(device, 9, lengths, 16, 2, 64, "f16")
    turned = PagedKvCache(cache.k_pages.transpose(1, 2).contiguous().transpose(1, 2), cache.v_pages.transpose(1, 2).contiguous().transpose(1, 2))
    rows = torch.randn((2 * tokens, 3 + 8 * 64), generator=g, device=device).half()
    q = rows[:, 3:3 + 4 * 64].view(2 * tokens, 4, 64)
    q0 = q.contiguous()
    out = _run(backend, device, cache, table, lengths, q0)
    _check(cache, table, lengths, q0, out)
    assert same_bits(out, _run(backend, device, turned, table, lengths, q))
    wide = torch.full((2 * tokens, 4, 70), 5.0, device=device, dtype=torch.float16)
    backend.gqa_attention_paged(q, cache, _i32(table, device), _i32(lengths, device), wide[..., 3:67])
    assert same_bits(wide[..., 3:67], out) and torch.all(wide[..., :3] == 5.0) and torch.all(wide[..., 67:] == 5.0)
    backend.gqa_attention_paged(q, cache, _i32(table, device), _i32(lengths, device), q)
    assert same_bits(q, out)
    wide_table = torch.full((2, table.shape[1] + 5), -1, device=device, dtype=torch.int32)
    wide_table[:, :table.shape[1]] = _i32(table, device)
    q2 = q0.clone()
    backend.gqa_attention_paged(q2, cache, wide_table[:, :table.shape[1]], _i32(lengths, device), q2, shared_pages=0)
    assert same_bits(q2, out)


def test_far_pages(backend, device):
    """Pages past 2^31 elements."""
    page, kvh, dim = 256, 8, 256
    pages = (1 << 31) // (page * kvh * dim) + 3
    cache = PagedKvCache.allocate(pages, kvh, page, dim, device=device)
    g = torch.Generator(device=device).manual_seed(1)
    table = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    for p in table[0]:
        cache.k_pages[int(p)].normal_(generator=g)
        cache.v_pages[int(p)].normal_(generator=g)
    small = PagedKvCache(cache.k_pages[table[0].tolist()], cache.v_pages[table[0].tolist()])
    for tokens in (1, 40):
        q = torch.randn((tokens, 8, dim), generator=g, device=device).half()
        out = _run(backend, device, cache, table, [700], q)
        assert same_bits(out, _run(backend, device, small, [[0, 1, 2]], [700], q))
        _check(small, np.array([[0, 1, 2]]), [700], q, out)


def test_wild_counts(backend, device):
    """cu_tokens that no program should give: nothing outside the operands is touched."""
    cache, table, g = _make(device, 3, [40, 40], 16, 2, 64, "f16")
    for cu in ([-5, 3, 900], [9, 2, 9], [0, 0, 0], [4, 4, 2]):
        q = torch.randn((9, 4, 64), generator=g, device=device).half()
        out = torch.full((11, 4, 64), 9.0, device=device, dtype=torch.float16)
        backend.gqa_attention_paged(q, cache, _i32(table, device), _i32([40, 40], device), out[1:10], cu_tokens=_i32(cu, device))
        assert torch.all(out[0] == 9.0) and torch.all(out[10] == 9.0)
