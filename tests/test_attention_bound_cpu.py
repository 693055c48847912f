"""The bounds that attention over long rows is held to reject a result that lost or repeated a tile.  The
mistakes are planted in the float64 restatement."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import attention_bound, step_ref


def _values(rng, tokens, kv_heads, dim, mean):
    x = rng.standard_normal((kv_heads, tokens, dim)) + rng.standard_normal((kv_heads, 1, dim)) * mean
    return step_ref.dequantize(*step_ref.quantize(x, 64))


@pytest.mark.parametrize("tokens,groups", [(36000, 512), (36000, 2), (20000, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_random_rows(tokens, groups, dim):
    rng = np.random.default_rng(dim + tokens)
    k, v = _values(rng, tokens, 1, dim, 1.5), _values(rng, tokens, 1, dim, 0.0)
    q = rng.standard_normal((3, dim))
    scale = dim ** -0.5 / 16
    want, mag, reach, peak = attention_bound.attention(q, k, v, scale)
    for info in (torch.finfo(torch.float16), torch.finfo(torch.bfloat16)):
        limit = attention_bound.bound(want, mag, reach, peak, tokens, *attention_bound.tiles_per_wave(groups, tokens), info)
        for tile in (0, 1, 255, 256, tokens // 64, tokens // 32 - 1):
            ids = range(32 * tile, 32 * tile + 32)
            for wrong in (dict(left_out=ids), dict(twice=ids)):
                got = attention_bound.attention(q, k, v, scale, **wrong)[0]
                assert np.any(np.abs(got - want) > limit), (tile, wrong.keys())


@pytest.mark.parametrize("tokens,dim", [(36000, 64), (36000, 128), (36000, 256), (131072, 128)])
def test_marked_tokens(tokens, dim):
    """... of marked tokens: one token lost, repeated, or taken for another."""
    at = attention_bound.marks(tokens, 2, dim, 1)
    seen = np.arange(tokens)
    want = attention_bound.marked(at, dim, seen)
    limit = attention_bound.marked_bound(want, torch.finfo(torch.float16))
    for t in (0, 31, 8191, 8192, tokens // 2, tokens - 1):
        for wrong in (np.delete(seen, t), np.append(seen, t), np.append(np.delete(seen, t), (t + 777) % tokens)):
            got = attention_bound.marked(at, dim, wrong)
            if len(wrong) == tokens and np.array_equal(got, want):      # the other token marks the same dims
                continue
            assert np.any(np.abs(got - want) > limit), t


def test_split_rule_is_covered():
    """A wave has at most 64 tiles up to four million tokens."""
    for groups in (1, 2, 16, 64, 255, 256, 511, 512, 4096):
        for tokens in (1, 700, 2048, 2080, 8192, 8193, 36000, 131072, 1 << 22):
            tiles, parts = attention_bound.tiles_per_wave(groups, tokens)
            assert tiles <= 64 and parts <= 513 and 4 * tiles * parts >= tokens // 32
