"""Float64 restatements, in numpy, of the operators on a paged KV cache, by their definitions, and
how far a result of attention may be from its restatement."""

from __future__ import annotations

import numpy as np
import torch


def np64(t):
    return t.double().cpu().numpy()


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def row_counts(cu, rows, tokens):
    return [cu[r + 1] - cu[r] for r in range(rows)] if cu is not None else [tokens // rows] * rows


def places(table, start, n, page):
    """(page id, slot) of positions start .. start + n - 1 of a row, (-1, 0) where there is none."""
    out = []
    for p in range(start, start + n):
        out.append((int(table[p // page]), p % page) if 0 <= p < len(table) * page else (-1, 0))
    return out


def attention(q, k_pages, v_pages, table, lengths, counts, page, *, window=0, sinks=None, scale=None, selected=None,
              max_length=None):
    """q [tokens, heads, D], pages [pages, kv_heads, page, D] float64.  Per query: the output, sum p |v|, the
    largest sum of |q| |k| scale, the tokens seen, the largest finite |v|."""
    tokens, heads, d = q.shape
    kvh = k_pages.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, mag, reach, seen = np.zeros_like(q), np.zeros_like(q), np.zeros((tokens, heads, 1)), np.zeros(tokens, dtype=int)
    at, peak = 0, np.zeros((tokens, heads, 1))
    for r, t in enumerate(counts):
        n = max(0, min(lengths[r], len(table[r]) * page, max_length or 1 << 30))
        for i in range(t):
            hi = n - (t - 1 - i)
            lo = max(0, hi - window) if window else 0
            for j in range(kvh):
                vis = np.arange(lo, max(lo, hi))
                if selected is not None:
                    chosen = [int(p) for p in selected[r][j] if 0 <= p < len(table[r])]
                    vis = np.concatenate([vis[vis // page == p] for p in chosen]) if chosen else vis[:0]
                seen[at + i] = max(seen[at + i], len(vis))
                if len(vis) == 0:
                    continue
                ids = np.asarray(table[r])[vis // page]
                bad = (ids < 0) | (ids >= len(k_pages))
                ids = np.where(bad, 0, ids)
                k, v = k_pages[ids, j, vis % page], v_pages[ids, j, vis % page]
                for h in range(j * heads // kvh, (j + 1) * heads // kvh):
                    s = np.where(bad, np.nan, k @ q[at + i, h] * scale)
                    top = s.max() if sinks is None else max(s.max(), sinks[h])
                    p = np.exp(s - top)
                    den = p.sum() + (0.0 if sinks is None else np.exp(sinks[h] - top))
                    out[at + i, h], mag[at + i, h] = p @ v / den, p @ np.abs(v) / den
                    peak[at + i, h] = np.abs(v[np.isfinite(v)]).max(initial=0.0)
                    reach[at + i, h] = (np.abs(k) @ np.abs(q[at + i, h])).max() * abs(scale)
        at += t
    return out, mag, reach, seen, peak


def attention_bound(want, mag, reach, seen, peak, dtype):
    """Scores: D exact products added in binary32 and one scaling, (D + 24) 2^-24 of the largest sum of
    |q| |k| scale; the exponential 2^-20 with the rounding of its argument.  Both count twice, above and below the
    line.  Weights: rounded once to the cache's 16-bit type, p' = p (1 + d) with |d| <= e = finfo.eps / 2, for the
    product with V and for their own sum alike: sum p' v / sum p' - out = (sum p d v - out sum p d) / sum p', no more
    than e (sum p |v| / sum p + |out|) / (1 - e); where that type is fp16 at least half of its smallest step,
    2^-25 of the largest weight for each token (weights are scaled so that the largest is no less than 1), times the
    largest |v|.
    Sums over the tokens seen: every token adds at most one rounding in each of two sums, 2^-24 of them, and a few
    dozen rescalings.  The store: half a step of the type."""
    info = torch.finfo(dtype)
    d = want.shape[-1]
    rel = 2 * ((d + 24) * 2.0 ** -24 * reach + 2.0 ** -20) + (2 * seen[:, None, None] + 64) * 2.0 ** -24 + info.eps / 2
    small = seen[:, None, None] * 2.0 ** -25 * peak if dtype == torch.float16 else 0.0
    rel, out = rel * (1 + 2.0 ** -7), info.eps * np.abs(want) * (1 + 2.0 ** -7)     # 1 / (1 - e); weights' sum and the store
    return rel * mag + small + out + info.tiny * info.eps


def scores(q, bounds, table_row, pages_of_row):
    """float32 scores [kv_heads, pages] of q [heads, D] and bounds [pages, kv_heads, 2, D], float64."""
    heads, kvh = q.shape[0], bounds.shape[1]
    out = np.zeros((kvh, pages_of_row), dtype=np.float32)
    for p in range(pages_of_row):
        i = int(table_row[p])
        for j in range(kvh):
            if not 0 <= i < len(bounds):
                out[j, p] = np.nan
                continue
            with np.errstate(invalid="ignore"):
                part = [np.float32(np.maximum(x * bounds[i, j, 0], x * bounds[i, j, 1]).sum())
                        for x in q[j * heads // kvh:(j + 1) * heads // kvh]]
            out[j, p] = np.max(part)
    return out


def select(score, count, first, last):
    """The pages kept of float32 scores [pages], ascending, -1 behind them."""
    pages = len(score)
    forced = set(range(min(first, pages))) | set(range(max(0, pages - last), pages))
    key = np.where(np.isnan(score), np.inf, score)
    free = sorted((p for p in range(pages) if p not in forced), key=lambda p: (not np.isnan(score[p]), -key[p], p))
    keep = sorted([*forced, *free[:max(0, count - len(forced))]])[:count]
    return keep + [-1] * (count - len(keep))


def scattered(rng, needs, pages, shared=0):
    """A table of distinct pages, in no order; what no token needs is -1.  The first `shared` are every row's."""
    order = rng.permutation(pages)
    width = max(max(needs, default=0), shared, 1)
    table, at = -np.ones((len(needs), width), dtype=np.int32), shared
    for r, n in enumerate(needs):
        table[r, :shared] = order[:shared]
        own = max(0, n - shared)
        table[r, shared:shared + own] = order[at:at + own]
        at += own
    return table
