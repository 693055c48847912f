"""Float64 attention over the 4-bit cache and how far a result may be from it, by the depth of the
kernel's additions rather than by the number of tokens.

Weights.  A score is a sum of dim exact products and three parts per group in binary32, scaled once,
with the running maximum taken off: (dim + 24) 2^-24 of the largest sum of |q| |k| times the scale, and
2^-20 for the exponential (2^-22) and the roundings of an exponent that is near 7.  It counts twice: above
and below the line of the quotient.

Sums.  A wave adds `tiles` tiles of 32 tokens in two products each (a weight is two fp16 parts), a
product at most eight times to its accumulator; its weights four times a tile.  Four waves and `parts`
workgroups are joined, each after a scaling.  So an output has at most 16 tiles + 4 tiles + 2 (4 +
parts) + 32 additions above and below the line, 2^-24 of sum p |v| each.  A weight's second part is cut
at 2^-21 of the weight, or at 2^-31 of the largest weight where that is more: for every token."""

from __future__ import annotations

import numpy as np


def tiles_per_wave(groups: int, tokens: int) -> tuple[int, int]:
    """(tiles of a wave, workgroups of a row) at most, for a call of `groups` (row, KV head, sixteen
    query heads) whose rows see up to `tokens`."""
    tiles = -(-tokens // 32) + 1
    if tiles <= 24 or (groups >= 256 and tiles <= 64):
        return -(-tiles // 4), 1
    fill = max(1, 512 // groups)
    share = min(256, -(-tiles // min(fill, -(-tiles // 8))))
    return -(-share // 4), -(-tiles // share)


def attention(q, k, v, scale, left_out=(), twice=()):
    """q [heads, D], k / v [kv_heads, tokens, D]: the output of all tokens but `left_out`, those of `twice`
    counted twice, and what the bound takes: sum p |v|, the largest sum of |q| |k| scale, and the largest
    share of one token times the largest |v|."""
    heads, kv, n = q.shape[0], k.shape[0], k.shape[1]
    count = np.ones(n)
    count[list(left_out)] = 0.0
    count[list(twice)] = 2.0
    out, mag = np.zeros_like(q), np.zeros_like(q)
    reach, peak = np.zeros((heads, 1)), np.zeros((heads, 1))
    for h in range(heads):
        kk, vv = k[h * kv // heads], v[h * kv // heads]
        s = kk @ q[h] * scale
        p = np.exp(s - s.max()) * count
        den = p.sum()
        out[h], mag[h] = p @ vv / den, p @ np.abs(vv) / den
        reach[h] = (np.abs(kk) @ np.abs(q[h])).max() * abs(scale)
        peak[h] = p.max() / den * np.abs(vv).max()
    return out, mag, reach, peak


def bound(want, mag, reach, peak, tokens, tiles, parts, info):
    """`info`: torch.finfo of the output's type."""
    dim = want.shape[1]
    weights = 2 * ((dim + 24) * 2.0 ** -24 * reach + 2.0 ** -20)
    sums = 2 * (20 * tiles + 2 * (4 + parts) + 32) * 2.0 ** -24 + 2.0 ** -21
    return (weights + sums) * mag + tokens * 2.0 ** -31 * peak + info.eps / 2 * np.abs(want) * (1 + 2.0 ** -10) + info.tiny * info.eps


# ------------------------------------------------------------------ every token visible
def marks(tokens: int, kv_heads: int, dim: int, seed: int):
    """The dim that a token marks in each KV head, [tokens, kv_heads]: with equal weights, values of 15 there
    and 0 elsewhere, an output is 15 times the tokens in sight that mark its dim, over all in sight."""
    return np.random.default_rng(seed).integers(0, dim, (tokens, kv_heads))


def marked(at, dim, seen):
    """Outputs [kv_heads, dim] for the tokens `seen` (indexes, twice if counted twice)."""
    out = np.zeros((at.shape[1], dim))
    for h in range(at.shape[1]):
        out[h] = 15.0 * np.bincount(at[seen, h], minlength=dim) / max(len(seen), 1)
    return out


def marked_bound(want, info):
    """All terms are whole numbers below 2^24 (weights of 2^7, codes of 15 at a step of 1), so the sums are
    exact: what is rounded is the quotient, to binary32 and to the output's type."""
    return np.abs(want) * (info.eps / 2 + 2.0 ** -22) + info.tiny * info.eps / 2
