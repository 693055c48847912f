"""Attention over pages by each of its kernels: batches with so many KV heads that short rows go to the kernel for many
columns, prefixes long enough to be computed once for the batch, either way, and selections for many query heads of a KV
head.  Against float64 within the bound that ``tests/paged_ref.py`` derives."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.paged_ref import same_bits
from tests.test_paged_attention_gpu import _DT, _RAGGED, _check, _i32, _make, _run
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window", [(40, 20, 64, 16, 0), (32, 16, 128, 64, 0), (48, 24, 128, 16, 40), (18, 6, 256, 32, 0),
                                                            (20, 20, 64, 256, 130)])
@pytest.mark.parametrize("sinks", [False, True])
def test_ragged_chunks(backend, device, dtype, heads, kv_heads, dim, page, window, sinks):
    counts, lengths = _RAGGED
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    cache, table, g = _make(device, heads + dim, lengths, page, kv_heads, dim, dtype)
    q = torch.randn((cu[-1] + 5, heads, dim), generator=g, device=device).to(_DT[dtype])
    kw = dict(window=window, sinks=torch.randn(heads, generator=g, device=device) * 2 if sinks else None)
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, cu, **kw), cu, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(70, 64, 32, 64), (40, 40, 20, 128), (33, 48, 24, 256)])
def test_as_many_tokens_for_every_row(backend, device, dtype, tokens, heads, kv_heads, dim):
    lengths = [tokens, tokens + 1, 200, 1, 0, 151, 64, 17]
    cache, table, g = _make(device, tokens, lengths, 16, kv_heads, dim, dtype)
    q = torch.randn((len(lengths) * tokens, heads, dim), generator=g, device=device).to(_DT[dtype])
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q))


@pytest.mark.parametrize("dim", [64, 128])
def test_bad_table_entries(backend, device, dim):
    counts, lengths = [90, 100, 40, 40], [100, 100, 100, 40]
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    cache, table, g = _make(device, 5, lengths, 16, 20, dim, "f16")
    q = torch.randn((cu[-1], 40, dim), generator=g, device=device).half()
    table[0, 1], table[1, 6], table[2, 0] = -1, cache.pages, 1 << 30
    for kw in (dict(), dict(window=30)):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, cu, **kw), cu, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_and_infinities_out_of_sight(backend, device, dtype, dim):
    counts, lengths = [130, 132], [180, 132]
    cu = [0, 130, 262]
    cache, table, g = _make(device, 6, lengths, 16, 20, dim, dtype)
    q = torch.randn((262, 40, dim), generator=g, device=device).to(_DT[dtype])
    clean = _run(backend, device, cache, table, lengths, q, cu, window=30)
    at = 115                                                  # of row 0: seen by its queries from 65 on
    page, slot = int(table[0, at // 16]), at % 16
    cache.v_pages[page, :, slot, 3] = float("nan")
    cache.v_pages[page, :, slot, 40] = float("inf")
    cache.k_pages[int(table[0, (at + 1) // 16]), 0, (at + 1) % 16, 5] = float("nan")
    out = _run(backend, device, cache, table, lengths, q, cu, window=30)
    _check(cache, table, lengths, q, out, cu, window=30)
    assert same_bits(out[:65], clean[:65]) and same_bits(out[130:], clean[130:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(144, 2, 64), (80, 2, 128), (40, 2, 256), (33, 1, 128)])
def test_selected_pages_of_many_heads(backend, device, dtype, heads, kv_heads, dim):
    """More query heads to a KV head than a workgroup takes."""
    page, count, lengths = 16, 6, [200, 0, 3, 7 * 16, 11 * 16 + 1]
    rng = np.random.default_rng(heads)
    cache, table, g = _make(device, heads, lengths, page, kv_heads, dim, dtype)
    sel = -np.ones((5, kv_heads, count), dtype=np.int32)
    for r, n in enumerate(lengths):
        for j in range(kv_heads):
            held = rng.permutation(-(-n // page) + 2)[:count]
            sel[r, j, count - len(held):] = held              # behind places of none
    q = torch.randn((5, heads, dim), generator=g, device=device).to(_DT[dtype])
    for kw in (dict(), dict(sinks=torch.randn(heads, generator=g, device=device))):
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, selected=sel, **kw), selected=sel, **kw)


def test_pages_at_the_end_of_long_selections(backend, device):
    """Selections much wider than a row has pages, with what they name at any place."""
    lengths, count = [16 * 70, 16 * 9, 40], 600
    cache, table, g = _make(device, 3, lengths, 16, 2, 64, "bf16")
    rng = np.random.default_rng(1)
    sel = -np.ones((3, 2, count), dtype=np.int32)
    for r, n in enumerate(lengths):
        for j in range(2):
            held = rng.permutation(-(-n // 16))
            sel[r, j, np.append(rng.permutation(count - 1)[:len(held) - 1], count - 1)] = held      # the last place too
    q = torch.randn((3, 8, 64), generator=g, device=device).bfloat16()
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, selected=sel), selected=sel)


def _prefix(device, rows, kv_heads, dim, page, shared, dtype, seed=0):
    base = shared * page
    lengths = [(base + 1, base, base - page - 3, 0, base + 77, 1, base + 3 * page, base - 1, base + 40)[r % 9] for r in range(rows)]
    cache, table, g = _make(device, rows + dim + seed, lengths, page, kv_heads, dim, dtype, shared)
    for p in table[0, :shared]:
        cache.k_pages[p] = torch.randn(cache.k_pages[p].shape, generator=g, device=device).to(cache.dtype)
        cache.v_pages[p] = torch.randn(cache.v_pages[p].shape, generator=g, device=device).to(cache.dtype)
    return cache, table, lengths, g


@pytest.mark.parametrize("rows,tokens,heads,kv_heads,dim,shared", [(40, 1, 8, 4, 256, 1000), (130, 1, 2, 2, 64, 4000), (24, 1, 20, 10, 128, 1000),
                                                                   (20, 2, 10, 5, 128, 1500)])
def test_prefix_in_blocks_of_columns(backend, device, rows, tokens, heads, kv_heads, dim, shared):
    page = 16 if dim == 256 else 64
    cache, table, lengths, g = _prefix(device, rows, kv_heads, dim, page, shared // page, "bf16")
    q = torch.randn((rows * tokens, heads, dim), generator=g, device=device).bfloat16()
    sinks = torch.randn(heads, generator=g, device=device)
    for kw in (dict(), dict(window=shared // 2 + 5, sinks=sinks)):
        kw["shared_pages"] = shared // page
        _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, **kw), **kw)


def test_prefix_of_ragged_rows(backend, device):
    counts = [1, 0, 3, 1, 2, 1, 1, 1, 4] * 3
    cache, table, lengths, g = _prefix(device, 27, 8, 128, 64, 20, "f16")
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    q = torch.randn((cu[-1] + 3, 16, 128), generator=g, device=device).half()
    out = _run(backend, device, cache, table, lengths, q, cu, shared_pages=20)
    _check(cache, table, lengths, q, out, cu)
    other = table.copy()
    other[1:, :20] = -1
    assert same_bits(out, _run(backend, device, cache, other, lengths, q, cu, shared_pages=20))


def test_prefix_by_the_kernel_for_many_columns(backend, device):
    """640 columns of a KV head behind 4992 tokens."""
    rows, shared = 160, 78
    cache, table, lengths, g = _prefix(device, rows, 8, 64, 64, shared, "bf16")
    q = torch.randn((rows * 4, 8, 64), generator=g, device=device).bfloat16()
    kw = dict(window=3003, sinks=torch.randn(8, generator=g, device=device))
    _check(cache, table, lengths, q, _run(backend, device, cache, table, lengths, q, shared_pages=shared, **kw), **kw)
    q = q[:rows].contiguous().repeat(2, 1, 1)
    out = _run(backend, device, cache, table, lengths, q, shared_pages=shared)
    other = table.copy()
    other[1:, :shared] = -1
    assert same_bits(out, _run(backend, device, cache, other, lengths, q, shared_pages=shared))


def test_ignored_sharing_reads_row_0s_entries(backend, device):
    """A short prefix, which every row reads for itself, from row 0's pages."""
    for tokens in (1, 50):
        cache, table, lengths, g = _prefix(device, 9, 2, 64, 16, 5, "f16")
        q = torch.randn((9 * tokens, 4, 64), generator=g, device=device).half()
        out = _run(backend, device, cache, table, lengths, q, shared_pages=5)
        _check(cache, table, lengths, q, out)
        other = table.copy()
        other[1:, :5] = -1
        assert same_bits(out, _run(backend, device, cache, other, lengths, q, shared_pages=5))


def test_the_same_call_gives_the_same_bits(backend, device):
    cache, table, lengths, g = _prefix(device, 27, 8, 128, 64, 20, "bf16", 1)
    counts = [1, 0, 3, 1, 2, 1, 1, 1, 300] * 3
    cu = np.concatenate(([0], np.cumsum(counts))).tolist()
    sel = torch.empty((27, 8, 9), device=device, dtype=torch.int32)
    one, chunk = (torch.randn((n, 16, 128), generator=g, device=device).bfloat16() for n in (27, cu[-1]))
    cache.k_bounds.normal_(generator=g)

    def run():
        backend.select_pages(one, cache, _i32(table, device), _i32(lengths, device), sel)
        return [sel.clone(), _run(backend, device, cache, table, lengths, one), _run(backend, device, cache, table, lengths, one, shared_pages=20),
                _run(backend, device, cache, table, lengths, chunk, cu, shared_pages=20),
                _run(backend, device, cache, table, lengths, one, selected=sel.cpu().numpy())]

    first = run()
    for _ in range(3):
        assert all(same_bits(a, b) for a, b in zip(first, run()))


def test_empty_batches(backend, device):
    """No rows, and a table without pages: nothing happens; tokens behind the last row stay."""
    cache, _, g = _make(device, 4, [20], 16, 2, 64, "f16")
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.k_bounds)]
    for width in (0, 3):
        for tokens in (0, 4):
            cu = _i32([0], device) if tokens else None
            table, none = _i32(np.zeros((0, width)), device), _i32([], device)
            q, kv = (torch.randn((tokens, h, 64), generator=g, device=device).half() for h in (4, 2))
            turned, out = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
            backend.rotary_append_paged(cache, q, kv, kv.clone(), table, none, None, turned, cu_tokens=cu)
            backend.gqa_attention_paged(q, cache, table, none, out, cu_tokens=cu)
            backend.select_pages(q[:0], cache, table, none, _i32(np.zeros((0, 2, 5)), device))
            assert torch.all(out == 9.0) and torch.all(turned == 9.0)
    assert all(same_bits(a, b) for a, b in zip(before, (cache.k_pages, cache.v_pages, cache.k_bounds)))


def test_a_table_that_is_a_column(backend, device):
    cache, table, g = _make(device, 5, [13, 16], 16, 2, 64, "f16")
    q, k, v = (torch.randn((2, h, 64), generator=g, device=device).half() for h in (4, 2, 2))
    plain = _run(backend, device, cache, table, [13, 16], q)
    column = torch.stack((_i32(table[:, 0], device), _i32([-1, -1], device)), 0).t()[:, :1]
    assert column.stride() == (1, 2)
    out = torch.empty_like(q)
    backend.gqa_attention_paged(q, cache, column, _i32([13, 16], device), out)
    assert same_bits(plain, out)
    backend.rotary_append_paged(cache, None, k, v, column, _i32([3, 9], device), None)
    for r, slot in enumerate((3, 9)):
        assert same_bits(cache.k_pages[int(table[r, 0]), :, slot], k[r]) and same_bits(cache.v_pages[int(table[r, 0]), :, slot], v[r])
    sel = backend.select_pages(q, cache, column, _i32([13, 0], device), _i32(np.zeros((2, 2, 2)), device), first_pages=0, last_pages=1)
    assert sel.tolist() == [[[0, -1]] * 2, [[-1, -1]] * 2]


def test_strided_operands_in_place(backend, device):
    """q as an odd part of a fused row, out in place and as a view, a cache with its tokens before its heads."""
    lengths, cu = [150, 131], [0, 130, 262]
    cache, table, g = _make(device, 9, lengths, 16, 20, 64, "f16")
    turned = PagedKvCache(cache.k_pages.transpose(1, 2).contiguous().transpose(1, 2), cache.v_pages.transpose(1, 2).contiguous().transpose(1, 2))
    rows = torch.randn((262, 3 + 48 * 64), generator=g, device=device).half()
    q = rows[:, 3:3 + 40 * 64].view(262, 40, 64)
    q0 = q.contiguous()
    out = _run(backend, device, cache, table, lengths, q0, cu)
    _check(cache, table, lengths, q0, out, cu)
    assert same_bits(out, _run(backend, device, turned, table, lengths, q, cu))
    wide = torch.full((262, 40, 70), 5.0, device=device, dtype=torch.float16)
    call = lambda to: backend.gqa_attention_paged(q, cache, _i32(table, device), _i32(lengths, device), to, cu_tokens=_i32(cu, device))  # noqa: E731
    call(wide[..., 3:67])
    assert same_bits(wide[..., 3:67], out) and torch.all(wide[..., :3] == 5.0) and torch.all(wide[..., 67:] == 5.0)
    call(q)
    assert same_bits(q, out)


def test_far_pages(backend, device):
    """Pages past 2^31 elements; more queries than tokens."""
    page, kvh, dim = 256, 8, 256
    pages = (1 << 31) // (page * kvh * dim) + 3
    cache = PagedKvCache.allocate(pages, kvh, page, dim, device=device)
    g = torch.Generator(device=device).manual_seed(1)
    table = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    for p in table[0]:
        cache.k_pages[int(p)].normal_(generator=g)
        cache.v_pages[int(p)].normal_(generator=g)
    small = PagedKvCache(cache.k_pages[table[0].tolist()], cache.v_pages[table[0].tolist()])
    q = torch.randn((1100, 8, dim), generator=g, device=device).half()
    out = _run(backend, device, cache, table, [700], q)
    assert same_bits(out, _run(backend, device, small, [[0, 1, 2]], [700], q)) and torch.all(out[:400] == 0)
    _check(small, np.array([[0, 1, 2]]), [700], q[-90:], out[-90:])


def test_wild_counts(backend, device):
    """cu_tokens that no program should give: nothing outside the operands is touched."""
    cache, table, g = _make(device, 3, [400, 400], 16, 20, 64, "f16")
    for cu in ([-5, 3, 900], [300, 2, 390], [0, 0, 0], [4, 4, 2], [200, 100, 400]):
        q = torch.randn((400, 40, 64), generator=g, device=device).half()
        out = torch.full((402, 40, 64), 9.0, device=device, dtype=torch.float16)
        backend.gqa_attention_paged(q, cache, _i32(table, device), _i32([400, 400], device), out[1:401], cu_tokens=_i32(cu, device))
        assert torch.all(out[0] == 9.0) and torch.all(out[401] == 9.0)
