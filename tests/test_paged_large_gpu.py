"""Attention over pages at sizes where work is split, ordered and joined, exactly: keys of 0 make all weights equal, and
token t's value is 1 in dim t % D and 0 elsewhere, so that a query that sees the tokens [lo, hi) gets, in dim d, the number
of them with t % D == d over hi - lo.  Counts and their sums are exact (weights are one power of two); the quotient
takes a division and a product in binary32 for each part and the store, 2^-8 + 2^-20 of it in bf16, 2^-11 + 2^-20 in fp16."""

from __future__ import annotations

import pytest
import torch

from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu


def _marked(device, lengths, page, kvh, dim, dtype, shared=0, seed=0):
    """A cache whose values mark their tokens, NaN where no row has any, and the table."""
    g = torch.Generator(device=device).manual_seed(seed)
    needs = [-(-n // page) for n in lengths]
    pages = shared + sum(max(0, n - shared) for n in needs) + 1
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    table = torch.full((len(lengths), max(max(needs), shared)), -1, device=device, dtype=torch.int32)
    cache = PagedKvCache.allocate(pages, kvh, page, dim, dtype, device=device)
    cache.v_pages.fill_(float("nan"))
    eye = torch.eye(dim, device=device, dtype=dtype)
    table[:, :shared] = order[:shared]
    at = shared
    for r, n in enumerate(needs):
        own = max(0, n - shared)
        table[r, shared:shared + own] = order[at:at + own]
        at += own
        for first, count in ((0, shared if r == 0 else 0), (shared, own)):
            ids = table[r, first:first + count].long()
            t = torch.arange(first * page, (first + count) * page, device=device)
            cache.v_pages[ids] = eye[t % dim].view(count, 1, page, dim).expand(count, kvh, page, dim)
    return cache, table, g


def _check(backend, device, lengths, counts, heads, kvh, dim, page, dtype, *, uniform=False, shared=0, window=0, seed=0, max_length=None):
    cache, table, g = _marked(device, lengths, page, kvh, dim, dtype, shared, seed)
    total = sum(counts)
    q = torch.randn((total, heads, dim), generator=g, device=device).to(dtype)
    cu = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], device=device, dtype=torch.int32)
    out = torch.full_like(q, float("nan"))
    backend.gqa_attention_paged(q, cache, table, torch.tensor(lengths, device=device, dtype=torch.int32), out, cu_tokens=None if uniform else cu,
                                shared_pages=shared, window=window, max_length=max_length)
    row = torch.repeat_interleave(torch.arange(len(counts), device=device), torch.tensor(counts, device=device))
    place = torch.arange(total, device=device) - cu.long()[row]
    hi = (torch.tensor(lengths, device=device)[row] - (torch.tensor(counts, device=device)[row] - 1 - place)).clamp_min(0)
    lo = (hi - window).clamp_min(0) if window else torch.zeros_like(hi)
    d = torch.arange(dim, device=device)
    upto = lambda x: (x[:, None] // dim + (d < x[:, None] % dim)).double()  # noqa: E731
    want = ((upto(hi) - upto(lo)) / (hi - lo).clamp_min(1)[:, None])[:, None]
    off = (out.double() - want).abs() - want * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)
    assert not torch.isnan(out).any()
    worst = off.amax((1, 2))
    assert worst.max() <= 0, (int(worst.argmax()), float(worst.max()), int((worst > 0).sum()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kvh,dim,page", [(40, 10, 128, 16), (32, 32, 64, 64), (16, 8, 256, 32), (24, 12, 128, 256)])
def test_chunks_of_uneven_prompts(backend, device, dtype, heads, kvh, dim, page):
    """More workgroups than run at once: long tiles first, heads dealt over the XCDs (whole ones and the rest)."""
    counts, lengths = [900, 1500, 0, 1, 1700, 33], [3000, 1500, 77, 2500, 1800, 3333]
    _check(backend, device, lengths, counts, heads, kvh, dim, page, dtype)


@pytest.mark.parametrize("heads,kvh,dim,tokens", [(16, 2, 128, 1024), (32, 8, 64, 1024), (8, 4, 256, 777), (8, 1, 64, 12), (30, 10, 128, 40), (16, 4, 64, 25)])
def test_as_many_queries_for_every_row(backend, device, heads, kvh, dim, tokens):
    _check(backend, device, [2049, tokens, 1300, 1900], [tokens] * 4, heads, kvh, dim, 32, torch.bfloat16, uniform=True)


@pytest.mark.parametrize("dim", [64, 128])
def test_more_rows_than_lanes(backend, device, dim):
    g = torch.Generator().manual_seed(dim)
    counts = torch.randint(0, 60, (150,), generator=g).tolist()
    lengths = [c + int(n) for c, n in zip(counts, torch.randint(0, 700, (150,), generator=g))]
    _check(backend, device, lengths, counts, 12, 4, dim, 16, torch.float16)
    _check(backend, device, lengths, counts, 12, 4, dim, 16, torch.float16, window=130)


@pytest.mark.parametrize("dim,window,tokens", [(64, 128, 900), (128, 100, 500), (256, 31, 300), (64, 1, 64), (128, 1000, 700)])
def test_windows_of_chunks(backend, device, dim, window, tokens):
    _check(backend, device, [4099, tokens, 1200], [tokens, tokens, tokens], 16, 2, dim, 32, torch.float16, uniform=True, window=window)
    _check(backend, device, [4099, 1200], [tokens, 7], 16, 2, dim, 32, torch.float16, window=window)


@pytest.mark.parametrize("dim,heads,kvh", [(64, 64, 8), (128, 40, 10), (256, 8, 2)])
@pytest.mark.parametrize("rows,length", [(48, 3000), (3, 20000), (300, 200)])
def test_single_tokens(backend, device, dim, heads, kvh, rows, length):
    lengths = [max(0, length - 61 * r) if r % 7 != 5 else r % 3 for r in range(rows)]
    _check(backend, device, lengths, [1] * rows, heads, kvh, dim, 64, torch.bfloat16, uniform=True)
    _check(backend, device, lengths, [1] * rows, heads, kvh, dim, 64, torch.bfloat16, uniform=True, window=500)


@pytest.mark.parametrize("page", [16, 256])
def test_one_row_of_many_tokens(backend, device, page):
    """Hundreds of parts of a query; a bound far above the length."""
    _check(backend, device, [200003], [1], 4, 1, 64, page, torch.float16, uniform=True)
    _check(backend, device, [70000], [3], 2, 1, 64, page, torch.bfloat16, uniform=True)


@pytest.mark.parametrize("dim,heads,kvh", [(64, 32, 8), (128, 16, 2), (256, 8, 2), (128, 10, 10)])
@pytest.mark.parametrize("rows,tokens", [(5, 1), (20, 1), (130, 1), (40, 4)])
def test_shared_prefix(backend, device, dim, heads, kvh, rows, tokens):
    """Few and many columns against the shared pages, with some rows that end inside them."""
    shared, page = 61, 16
    base = shared * page
    lengths = [base - 300 if r % 9 == 4 else 0 if r % 9 == 7 else base + 3 * r + tokens for r in range(rows)]
    _check(backend, device, lengths, [tokens] * rows, heads, kvh, dim, page, torch.bfloat16, uniform=True, shared=shared)


def test_long_shared_prefix(backend, device):
    lengths = [33000 + 11 * r for r in range(24)]
    _check(backend, device, lengths, [1] * 24, 64, 8, 128, 64, torch.bfloat16, uniform=True, shared=512)
    _check(backend, device, lengths, [3, 0, 200, 1] * 6, 16, 2, 64, 64, torch.float16, shared=512)


def test_a_bound_on_lengths(backend, device):
    """A table much wider than the rows need, planned for all of it and for less."""
    lengths = [500, 33, 1200, 0]
    for limit in (None, 1200, 4096):
        _check(backend, device, lengths, [1] * 4, 16, 2, 128, 16, torch.bfloat16, uniform=True, max_length=limit)


@pytest.mark.parametrize("kvh,window", [(16, 0), (32, 5)])
def test_most_rows_and_the_widest_table(backend, device, kvh, window):
    """65535 rows and tables of 2^30 - 256 tokens, which all rows share: by themselves and, with a window,
    by the kernel for few columns.  Slot t holds t + 1, and an odd number of tokens are seen: the mean is exact."""
    rows, pages = 65535, (1 << 22) - 1
    cache = PagedKvCache.allocate(1, kvh, 256, 64, device=device)
    cache.v_pages.copy_(torch.arange(1, 257, device=device)[:, None])
    table = torch.zeros((1, pages), device=device, dtype=torch.int32).expand(rows, pages)
    lengths = 1 + 2 * (torch.arange(rows, device=device, dtype=torch.int32) % 100)
    q = torch.ones((rows, kvh, 64), device=device, dtype=torch.float16)
    out = torch.full_like(q, float("nan"))
    backend.gqa_attention_paged(q, cache, table, lengths, out, window=window, shared_pages=pages if window else 0)
    want = (lengths + (lengths - window).clamp_min(0) + 1) / 2 if window else (lengths + 1) / 2
    assert int((out != want.half()[:, None, None]).sum()) == 0


def test_most_heads_of_a_kv_head_behind_many_tokens(backend, device):
    """65535 query heads of one KV head, with 2^23 + 2^18 tokens in one row and few in three: the longest column tiles begin
    first.  Values are 1 and 3 in turn, so the mean of an even number is exact."""
    heads, lengths = 65535, [256, (1 << 23) + (1 << 18), 2, 258]
    cache = PagedKvCache.allocate(1, 1, 256, 64, device=device)
    cache.v_pages.copy_(1 + 2 * (torch.arange(256, device=device) % 2)[:, None])
    table = torch.zeros((4, max(lengths) // 256), device=device, dtype=torch.int32)
    q = torch.ones((4, heads, 64), device=device, dtype=torch.float16)
    out = torch.full_like(q, float("nan"))
    backend.gqa_attention_paged(q, cache, table, torch.tensor(lengths, device=device, dtype=torch.int32), out)
    assert (out != 2).sum((1, 2)).tolist() == [0, 0, 0, 0]
