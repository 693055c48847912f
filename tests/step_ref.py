"""Float64 restatements, in numpy, of the operators of a decode step around its weights
(rotary positions, the 4-bit KV cache, attention over it, sampling), by their definitions."""

from __future__ import annotations

import numpy as np


# ------------------------------------------------------------------ rotary
def rotary(x, positions, inv_freq, interleaved, amplitude):
    """x [tokens, heads, dim] float64 -> the same, rotated."""
    r = 2 * len(inv_freq)
    out = x.astype(np.float64).copy()
    ang = np.asarray(positions, dtype=np.float64)[:, None] * inv_freq
    c, s = np.cos(ang)[:, None] * amplitude, np.sin(ang)[:, None] * amplitude
    ia, ib = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
    a, b = out[..., ia].copy(), out[..., ib].copy()
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


# ------------------------------------------------------------------ the 4-bit cache
def steps():
    """Every step that the format has, in increasing order: seven significant bits, multiples of
    2^-24, at most 4064."""
    v = {n * 2.0 ** e for e in range(-24, 7) for n in range(1, 129)}
    return np.array(sorted(x for x in v if x <= 4064.0))


_STEPS = steps()


def quantize(x, group):
    """x [..., D] float64 -> (codes [..., D], s, m [..., D / group]); NaN s and m for groups that
    are not finite."""
    g = np.asarray(x, dtype=np.float64).reshape(x.shape[:-1] + (-1, group))
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    m = np.clip(g.min(-1), -65504.0, 65504.0).astype(np.float16).astype(np.float64)
    reach = g.max(-1) - m
    at = np.searchsorted(15.0 * _STEPS, reach)          # first with 15 s >= reach
    s = np.where(reach > 0, _STEPS[np.minimum(at, len(_STEPS) - 1)], 0.0)
    y = np.divide(g - m[..., None], s[..., None], out=np.zeros_like(g), where=s[..., None] > 0)
    codes = np.clip(np.rint(y), 0, 15).astype(np.int64)
    s, m = np.where(bad, np.nan, s), np.where(bad, np.nan, m)
    codes = np.where(bad[..., None], 0, codes)
    return codes.reshape(x.shape), s, m


def dequantize(codes, s, m):
    group = codes.shape[-1] // s.shape[-1]
    return codes * np.repeat(s, group, -1) + np.repeat(m, group, -1)


def unpack_k(words):
    w = np.asarray(words).view(np.uint32)
    return np.stack([(w >> (4 * i)) & 15 for i in range(8)], -1).reshape(w.shape[:-1] + (-1,)).astype(np.int64)


def unpack_v(words):
    """[..., blocks, D] -> [..., tokens, D]"""
    w = np.asarray(words).view(np.uint32)
    t = np.stack([(w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15 for i in range(8)], -2)
    return t.reshape(w.shape[:-2] + (-1, w.shape[-1])).astype(np.int64)


def unpack_v_scales(vs):
    """[..., blocks, groups, 2, 8] -> s, m [..., tokens, groups]"""
    a = np.moveaxis(np.asarray(vs, dtype=np.float64), -1, -3)          # [..., blocks, 8, groups, 2]
    a = a.reshape(a.shape[:-4] + (-1,) + a.shape[-2:])
    return a[..., 0], a[..., 1]


# ------------------------------------------------------------------ attention
def attention(q, k, v, length, window=0, first=0, sinks=None, scale=None):
    """q [heads, D], k / v [kv_heads, tokens, D] float64; (out, sum of p |v|, largest sum of
    |q||k| scale, tokens seen)."""
    heads, d = q.shape
    kv = k.shape[0]
    n = max(0, min(length, k.shape[1]))
    t = np.arange(n)
    if window > 0:
        t = t[(t >= n - window) | (t < first)]
    scale = d ** -0.5 if scale is None else scale
    out, mag, reach = np.zeros((heads, d)), np.zeros((heads, d)), np.zeros((heads, 1))
    if len(t) == 0:
        return out, mag, reach, 0
    for h in range(heads):
        kk, vv = k[h * kv // heads][t], v[h * kv // heads][t]
        s = kk @ q[h] * scale
        top = s.max() if sinks is None else max(s.max(), sinks[h])
        p = np.exp(s - top)
        den = p.sum() + (0.0 if sinks is None else np.exp(sinks[h] - top))
        out[h], mag[h] = p @ vv / den, p @ np.abs(vv) / den
        reach[h] = (np.abs(kk) @ np.abs(q[h])).max() * abs(scale)
    return out, mag, reach, len(t)


# ------------------------------------------------------------------ sampling
def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, share) of one row of float64 logits."""
    x = np.asarray(x, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, 0.0
    top = x[order[0]]
    if not temperature > 0:
        order = order[:1]
        w = np.ones(1)
    else:
        with np.errstate(invalid="ignore"):
            w = np.where(x[order] == top, 1.0, np.exp(-(top - x[order]) / temperature))
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        w = w[: 1 + int(np.searchsorted(np.cumsum(w), max(top_p, 0.0) * np.cumsum(w)[-1]))]
    if min_p > 0:
        w = w[: max(1, int(np.count_nonzero(w >= min_p)))]
    cum = np.cumsum(w)
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    j = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(w) - 1)
    return int(order[j]), w[j] / cum[-1]
