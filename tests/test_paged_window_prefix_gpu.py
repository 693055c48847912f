"""A window together with shared pages that are computed once: rows whose window begins behind the prefix, beside rows that
still see its end.  What such a row does not see changes nothing of its result, however large its scores are there.
Against float64 within the bound that ``tests/paged_ref.py`` derives."""

from __future__ import annotations

import pytest
import torch

from tests.paged_ref import same_bits
from tests.test_paged_attention_gpu import _DT, _check, _make, _run

pytestmark = pytest.mark.gpu

# rows, tokens of each, heads, KV heads, head_dim, page, prefix (tokens), window: the prefix by the kernel for few columns, with
# one token a row and several, and by that for many
_CASES = [(16, 1, 32, 8, 64, 64, 8192, 4096), (20, 2, 10, 5, 128, 64, 2048, 1300), (40, 1, 8, 4, 256, 16, 2048, 1200),
          (64, 1, 64, 8, 128, 64, 8192, 2500), (160, 4, 8, 8, 64, 64, 4992, 3003), (64, 1, 32, 4, 256, 64, 4096, 3000)]


def _rows(device, case, dtype):
    """Every eighth row is far past the prefix, the others end up to half a window behind it; queries of the far rows have
    60 in their first dim and 1 in the second, of the others 0 and -1."""
    rows, tokens, heads, kv_heads, dim, page, base, window = case
    lengths = [base + window + tokens + r if r % 8 == 3 else base + tokens + 7 * r % (window // 2) for r in range(rows)]
    cache, table, g = _make(device, rows + dim, lengths, page, kv_heads, dim, dtype, base // page)
    for p in table[0, :base // page]:
        cache.k_pages[p].normal_(generator=g)
        cache.v_pages[p].normal_(generator=g)
    q = torch.randn((rows, tokens, heads, dim), generator=g, device=device).to(_DT[dtype])
    far = torch.arange(rows, device=device) % 8 == 3
    q[far, ..., 0], q[far, ..., 1] = 60.0, 1.0
    q[~far, ..., 0], q[~far, ..., 1] = 0.0, -1.0
    return cache, table, lengths, q.flatten(0, 1), far.repeat_interleave(tokens)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", _CASES)
def test_large_scores_out_of_sight(backend, device, case, dtype):
    """Scores of the prefix's last tokens that lie hundreds above those of the tokens that the far rows see."""
    cache, table, lengths, q, far = _rows(device, case, dtype)
    page, base, window = case[5:]
    kw = dict(window=window, shared_pages=base // page)
    clean = _run(backend, device, cache, table, lengths, q, **kw)
    cache.k_pages[table[0, base // page - 1], ..., 0] = 60.0
    out = _run(backend, device, cache, table, lengths, q, **kw)
    _check(cache, table, lengths, q, out, **kw)
    assert same_bits(out[far], clean[far])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", _CASES)
def test_infinite_keys_out_of_sight(backend, device, case, dtype):
    """An infinite key: a score of infinity for the far rows, which do not see it, and of minus infinity for the others."""
    cache, table, lengths, q, far = _rows(device, case, dtype)
    page, base, window = case[5:]
    kw = dict(window=window, shared_pages=base // page)
    clean = _run(backend, device, cache, table, lengths, q, **kw)
    cache.k_pages[table[0, base // page - 1], :, page - 5, 1] = float("inf")
    out = _run(backend, device, cache, table, lengths, q, **kw)
    assert same_bits(out[far], clean[far]) and torch.isfinite(out).all()
