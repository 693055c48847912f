"""cu_tokens that no program should give to the operators on a paged cache.  Values outside 0 .. tokens count as the nearest
inside: results are those of the clamped counts.  Counts that decrease give rows that are not defined; nothing outside the
cache and the output is touched, and what no row owns is left as it was."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.paged_ref import scattered
from tests.test_paged_append_gpu import _check as _check_append
from tests.test_paged_append_gpu import _copy, _inv_freq, _junk, _operands
from tests.test_paged_attention_gpu import _check as _check_attention
from tests.test_paged_attention_gpu import _i32, _make
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu

# more than 64 rows are looked for in another way
_MANY = [-3, -1, *range(0, 136, 2), 500]
_OUTSIDE = [[-5, 3, 900], [0, 0, 0], [-9, -2, 0], [2, 2, 7], [0, 4, 1 << 30], [-(1 << 31), 0, 9], _MANY]


def _call_append(backend, device, cache, q, k, v, out, table, starts, cu, f):
    backend.rotary_append_paged(cache, q, k, v, torch.from_numpy(table).to(device), _i32(starts, device), f, out, cu_tokens=_i32(cu, device))


@pytest.mark.parametrize("cu", _OUTSIDE)
@pytest.mark.parametrize("shift", [0, 1])                     # 1: operands off 16-byte boundaries
@pytest.mark.parametrize("bounds", [False, True])
def test_append_clamps_counts(backend, device, cu, shift, bounds):
    rows, tokens = len(cu) - 1, 200 if cu is _MANY else 9
    cache = PagedKvCache.allocate(3 * rows + 1, 2, 16, 64, bounds=bounds, device=device)
    _junk(cache, 1)
    before = _copy(cache)
    q, k, v = _operands(device, 4, tokens, 3, 2, 64, torch.float16)
    if shift:
        wide = torch.zeros((tokens, 3, 66), device=device, dtype=torch.float16)
        wide[..., 1:65] = q
        q = wide[..., 1:65]
    table = scattered(np.random.default_rng(1), [3] * rows, 3 * rows + 1)
    starts, out = [(5 * r) % 20 for r in range(rows)], torch.full((tokens, 3, 64), 9.0, device=device, dtype=torch.float16)
    f = _inv_freq(64, device)
    _call_append(backend, device, cache, q, k, v, out, table, starts, cu, f)
    clamped = np.clip(cu, 0, tokens).tolist()
    _check_append(backend, cache, before, q, k, v, out, table, starts, clamped, f, q_before=torch.full_like(out, 9.0))


@pytest.mark.parametrize("cu,owned", [([9, 2, 9], range(2, 9)), ([4, 4, 2], ()), ([6, 3, 0], ()), ([3, 8, 5], range(3, 8))])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_with_counts_that_decrease(backend, device, cu, owned, shift):
    stores = [torch.full((8, 2, 16, 64), 3.0, device=device, dtype=torch.float16) for _ in range(2)]
    marks = torch.full((8, 2, 2, 64), 3.0, device=device, dtype=torch.float16)
    cache = PagedKvCache(stores[0][1:7], stores[1][1:7], marks[1:7])
    q, k, v = _operands(device, 4, 9, 3, 2, 64, torch.float16)
    store = torch.full((11, 3, 64 + shift), 9.0, device=device, dtype=torch.float16)
    out = store[1:10, :, shift:]
    _call_append(backend, device, cache, q, k, v, out, np.array([[0, 5], [2, 3]], dtype=np.int32), [0, 12], cu, None)
    others = [i for i in range(9) if i not in owned]
    assert torch.all(out[others] == 9.0) and torch.all(store[[0, 10]] == 9.0) and torch.all(store[..., :shift] == 9.0)
    for t in (*stores, marks):
        assert torch.all(t[[0, 7]] == 3.0)
    if not owned:
        assert all(torch.all(t == 3.0) for t in (*stores, marks))


@pytest.mark.parametrize("cu", _OUTSIDE)
@pytest.mark.parametrize("heads,kv_heads,length", [(4, 2, 40), (40, 20, 60), (4, 1, 3000)])      # few columns, many, several parts
def test_attention_clamps_counts(backend, device, cu, heads, kv_heads, length):
    rows, tokens = len(cu) - 1, 200 if cu is _MANY else 9
    lengths = [length - r % 7 if r < 4 else 30 + r for r in range(rows)]
    cache, table, g = _make(device, heads, lengths, 16, kv_heads, 64, "f16")
    q = torch.randn((tokens, heads, 64), generator=g, device=device).half()
    store = torch.full((tokens + 2, heads, 64), 9.0, device=device, dtype=torch.float16)
    out = store[1:-1]
    backend.gqa_attention_paged(q, cache, _i32(table, device), _i32(lengths, device), out, cu_tokens=_i32(cu, device))
    assert torch.all(store[0] == 9.0) and torch.all(store[-1] == 9.0)
    _check_attention(cache, table, lengths, q, out, np.clip(cu, 0, tokens).tolist())


@pytest.mark.parametrize("cu,owned", [([9, 2, 9], range(2, 9)), ([4, 4, 2], ()), ([6, 3, 0], ()), ([3, 8, 5], range(3, 8))])
@pytest.mark.parametrize("heads,kv_heads,length", [(4, 2, 40), (40, 20, 60), (4, 1, 3000)])
def test_attention_with_counts_that_decrease(backend, device, cu, owned, heads, kv_heads, length):
    cache, table, g = _make(device, heads, [length, length - 3], 16, kv_heads, 64, "f16")
    q = torch.randn((9, heads, 64), generator=g, device=device).half()
    out = torch.full_like(q, 9.0)
    backend.gqa_attention_paged(q, cache, _i32(table, device), _i32([length, length - 3], device), out, cu_tokens=_i32(cu, device))
    assert torch.all(out[[i for i in range(9) if i not in owned]] == 9.0)
