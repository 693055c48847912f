"""The 4-bit KV cache: packing and reading back bit for bit against the format's definition, and
attention over it against float64.

Attention's error: scores are sums of D exact products and three parts per group in binary32, so a
score is off by at most (D + 16) 2^-24 times the largest sum of |q| |k| (q itself keeps 2^-31 of its
largest element); that is the relative error of a weight, twice in the quotient.  Weights are split to
2^-22 of themselves, the exponential and the running rescales add a few 2^-23, and sums of N weights N
2^-24 at most.  All of it times sum p |v|; the store adds half a step of its type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref
from thintensor_amd.kv_cache import Int4KvCache

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _np(t):
    return t.double().cpu().numpy()


def _held(cache, b):
    """Sequence b's K and V values and validity by definition, from the cache's own tensors."""
    ck = step_ref.unpack_k(cache.k_codes[b].cpu().numpy())
    ks = _np(cache.k_scales[b])
    cv = step_ref.unpack_v(cache.v_codes[b].cpu().numpy())
    vs, vm = step_ref.unpack_v_scales(cache.v_scales[b].cpu().numpy())
    return (ck, ks[..., 0], ks[..., 1]), (cv, vs, vm)


def _junk(cache, seed):
    """Contents that nothing may use: every bit pattern, NaN steps among them."""
    g = torch.Generator(device=cache.device).manual_seed(seed)
    for t in (cache.k_codes, cache.v_codes):
        t.copy_(torch.randint(-(2 ** 31), 2 ** 31, t.shape, generator=g, device=t.device))
    for t in (cache.k_scales, cache.v_scales):
        t.view(torch.int16).copy_(torch.randint(-(2 ** 15), 2 ** 15, t.shape, generator=g, device=t.device))
        t.masked_fill_(torch.rand(t.shape, generator=g, device=t.device) < 0.3, float("nan"))


def _same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _check_rows(cache, before, k, v, starts, counts):
    """The cache holds exactly what the definition packs, and `before` elsewhere."""
    for b in range(cache.batch):
        want = {"k": _held(before, b)[0], "v": _held(before, b)[1]}
        got = {"k": _held(cache, b)[0], "v": _held(cache, b)[1]}
        if b < k.shape[0]:
            for t in range(min(int(counts[b]), k.shape[1])):
                pos = int(starts[b]) + t
                if 0 <= pos < cache.capacity:
                    for n, x in (("k", k), ("v", v)):
                        c, s, m = step_ref.quantize(_np(x[b, t]), cache.group_size)
                        want[n][0][:, pos], want[n][1][:, pos], want[n][2][:, pos] = c, s, m
        for n in ("k", "v"):
            for a, w in zip(got[n], want[n]):
                assert np.array_equal(a, w, equal_nan=a.dtype.kind == "f"), (b, n)


_SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,group", _SHAPES)
def test_append_and_read(backend, device, dtype, dim, group):
    g = torch.Generator(device=device).manual_seed(dim + group)
    dt = _DT[dtype]
    cache = Int4KvCache.allocate(5, 3, 64, dim, group, device)
    _junk(cache, dim * group)
    starts = torch.tensor([0, 13, 60, -3], device=device, dtype=torch.int32)      # the cache's fifth sequence stays
    counts = torch.tensor([19, 8, 19, 7], device=device, dtype=torch.int32)
    before = Int4KvCache(cache.k_codes.clone(), cache.k_scales.clone(), cache.v_codes.clone(), cache.v_scales.clone())
    k = (torch.randn((4, 19, 3, dim), generator=g, device=device) * 3 + 1).to(dt)
    v = torch.randn((4, 19, 3, dim), generator=g, device=device).to(dt)
    v[0, 3] = 0.75                                                                # a constant group: no step
    v[1, 2] = torch.arange(dim, device=device).to(dt) * 0.5                       # ties between codes
    k[1, 2] = (torch.arange(dim, device=device) % 31).to(dt) * 0.25
    backend.kv_append_int4(cache, k, v, starts, counts)
    _check_rows(cache, before, k, v, starts, counts)
    for out in ("f16", "bf16", "f32"):
        ko, vo = (torch.full(k.shape, 77.0, device=device, dtype=_DT[out]) for _ in range(2))
        backend.kv_read_int4(cache, ko, vo, starts, counts)
        for n, o in (("k", ko), ("v", vo)):
            for b in range(4):
                held = dict(zip("kv", _held(cache, b)))[n]
                for t in range(19):
                    pos = int(starts[b]) + t
                    if t < int(counts[b]) and 0 <= pos < 64:
                        value = step_ref.dequantize(held[0][:, pos], held[1][:, pos], held[2][:, pos])
                        want = torch.from_numpy(value).float().to(_DT[out])
                        assert torch.equal(o[b, t].cpu().nan_to_num(1e9), want.nan_to_num(1e9)), (n, b, t)
                    else:
                        assert torch.all(o[b, t] == 77.0)


def test_append_one_by_one_equals_at_once(backend, device):
    g = torch.Generator(device=device).manual_seed(5)
    k, v = (torch.randn((2, 37, 2, 128), generator=g, device=device).half() for _ in range(2))
    a, b = (Int4KvCache.allocate(2, 2, 64, 128, 64, device) for _ in range(2))
    start = torch.tensor([3, 6], device=device, dtype=torch.int32)
    backend.kv_append_int4(a, k, v, start)
    for t in range(37):
        backend.kv_append_int4(b, k[:, t], v[:, t], start + t)
    assert all(_same_bits(x, y) for x, y in ((a.k_codes, b.k_codes), (a.k_scales, b.k_scales), (a.v_codes, b.v_codes),
                                             (a.v_scales, b.v_scales)))
    backend.kv_append_int4(b, k[:, 5], v[:, 5], start + 5)          # the same position again
    assert _same_bits(a.v_codes, b.v_codes)


def test_append_extreme_groups(backend, device):
    """Infinities, NaN, the largest and smallest values, wide ranges, -0."""
    dim = 64
    rows = torch.zeros((1, 12, 1, dim), device=device)
    g = torch.Generator(device=device).manual_seed(9)
    rows += torch.randn(rows.shape, generator=g, device=device)
    rows[0, 0, 0, 3] = float("inf")
    rows[0, 1, 0, 40] = float("nan")
    rows[0, 2] = 65504.0
    rows[0, 3, 0, :8] = torch.tensor([-65504.0, 65504.0] * 4, device=device)
    rows[0, 4] *= 2.0 ** -20
    rows[0, 5] = torch.where(rows[0, 5] > 0, 2.0 ** -24, -(2.0 ** -24))
    rows[0, 6, 0, 0] = 30000.0
    rows[0, 7] = -0.0
    rows[0, 8, 0, :4] = float("-inf")
    rows[0, 9] = torch.where(rows[0, 9] > 0, 7.5, -(2.0 ** -24))      # 15 steps and a little more
    starts = torch.zeros(1, device=device, dtype=torch.int32)
    for dt in (torch.float16, torch.bfloat16, torch.float32):
        x = rows.clone()
        if dt != torch.float16:
            x[0, 10, 0, :2] = torch.tensor([1e30, -1e30], device=device)
            x[0, 11, 0, :2] = torch.tensor([1e-30, -1e-38], device=device)
        x = x.to(dt)
        cache = Int4KvCache.allocate(1, 1, 32, dim, 32, device)
        before = Int4KvCache.allocate(1, 1, 32, dim, 32, device)
        backend.kv_append_int4(cache, x, x, starts)
        _check_rows(cache, before, x, x, starts, [12])
        ko, vo = torch.empty_like(x), torch.empty_like(x)
        backend.kv_read_int4(cache, ko, vo, starts)
        assert torch.isnan(ko[0, 0, 0, :32]).all() and torch.isfinite(ko[0, 0, 0, 32:]).all()
        assert torch.isnan(vo[0, 1, 0, 32:]).all() and torch.isnan(vo[0, 8, 0, :32]).all()
        assert torch.equal(ko.nan_to_num(3.0), vo.nan_to_num(3.0))


def test_append_strided_parts_of_qkv(backend, device):
    """k and v as views of a QKV row, a cache as a view of a larger one."""
    g = torch.Generator(device=device).manual_seed(11)
    qkv = torch.randn((6, 1 + (4 + 2 + 2) * 64), generator=g, device=device).half()
    whole = Int4KvCache.allocate(9, 2, 32, 64, 32, device)
    part = whole.sequences(2, 8)
    k = qkv[:, 1 + 4 * 64:1 + 6 * 64].view(6, 2, 64)
    v = qkv[:, 1 + 6 * 64:].view(6, 2, 64)
    starts = torch.arange(6, device=device, dtype=torch.int32)
    before = Int4KvCache.allocate(6, 2, 32, 64, 32, device)
    backend.kv_append_int4(part, k, v, starts)
    _check_rows(part, before, k[:, None], v[:, None], starts, [1] * 6)
    assert torch.count_nonzero(whole.k_codes[:2]) == 0 and torch.count_nonzero(whole.v_scales[8]) == 0


# ------------------------------------------------------------------ attention
def _filled(backend, device, batch, kv_heads, capacity, dim, group, seed, lengths):
    """A cache with `lengths` tokens of each sequence packed, junk behind them."""
    g = torch.Generator(device=device).manual_seed(seed)
    cache = Int4KvCache.allocate(batch, kv_heads, capacity, dim, group, device)
    _junk(cache, seed)
    n = max(max(lengths), 1)
    k = torch.randn((batch, n, kv_heads, dim), generator=g, device=device)
    k += torch.randn((1, 1, kv_heads, dim), generator=g, device=device) * 1.5
    v = torch.randn((batch, n, kv_heads, dim), generator=g, device=device)
    backend.kv_append_int4(cache, k, v, torch.zeros(batch, device=device, dtype=torch.int32),
                           torch.tensor(lengths, device=device, dtype=torch.int32))
    return cache, g


def _check_attention(cache, q, out, lengths, window=0, first=0, sinks=None, scale=None):
    dim = q.shape[-1]
    info = torch.finfo(q.dtype)
    for b, n in enumerate(lengths):
        (ck, ks, km), (cv, vs, vm) = _held(cache, b)
        n = max(0, min(n, cache.capacity))
        k, v = (step_ref.dequantize(c[:, :n], s[:, :n], m[:, :n]) for c, s, m in ((ck, ks, km), (cv, vs, vm)))
        want, mag, reach, seen = step_ref.attention(_np(q[b]), k, v, n, window, first,
                                                    None if sinks is None else _np(sinks), scale)
        got = _np(out[b])
        rel = 2 * (dim + 16) * 2.0 ** -24 * reach + (seen + 64) * 2.0 ** -24 + 2.0 ** -20
        bound = rel * mag + info.eps / 2 * np.abs(want) * (1 + 2.0 ** -10) + info.tiny * info.eps
        err = np.abs(got - want)
        assert np.all(err <= bound), (b, n, float((err - bound).max()), float(err.max()))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,group", _SHAPES)
def test_attention_shapes(backend, device, dtype, dim, group):
    lengths = [1, 33, 0, 200, 64]
    cache, g = _filled(backend, device, 5, 2, 224, dim, group, dim + group, lengths)
    q = torch.randn((5, 8, dim), generator=g, device=device).to(_DT[dtype])
    out = torch.full_like(q, 9.0)
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    backend.gqa_attention_int4(q, cache, out, n)
    assert torch.count_nonzero(out[2]) == 0
    _check_attention(cache, q, out, lengths)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (10, 2), (15, 1), (16, 1), (34, 2), (64, 1), (96, 3)])
def test_attention_head_layouts(backend, device, heads, kv_heads):
    lengths = [131, 47]
    cache, g = _filled(backend, device, 2, kv_heads, 160, 64, 32, heads, lengths)
    q = torch.randn((2, heads, 64), generator=g, device=device).half()
    sinks = torch.randn(heads, generator=g, device=device)
    for sk in (None, sinks, sinks.half(), sinks.bfloat16()):
        out = torch.empty_like(q)
        backend.gqa_attention_int4(q, cache, out, torch.tensor(lengths, device=device, dtype=torch.int32), sinks=sk, scale=0.2)
        _check_attention(cache, q, out, lengths, sinks=sk, scale=0.2)


@pytest.mark.parametrize("window,first", [(1, 0), (7, 0), (32, 1), (33, 4), (64, 64), (100, 33), (128, 4), (500, 10), (1000, 0),
                                          (2, 1000)])
def test_attention_windows(backend, device, window, first):
    lengths = [1, 2, 31, 32, 65, 129, 300, 640, 0]
    cache, g = _filled(backend, device, 9, 2, 640, 64, 32, window + first, lengths)
    q = torch.randn((9, 8, 64), generator=g, device=device).bfloat16()
    sinks = torch.randn(8, generator=g, device=device)
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    out = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, out, n, window=window, first_tokens=first, sinks=sinks)
    _check_attention(cache, q, out, lengths, window, first, sinks)


@pytest.mark.parametrize("dim,rows,kv_heads,heads", [(64, 64, 8, 24), (128, 64, 8, 8), (256, 70, 4, 16), (128, 33, 1, 48)])
def test_attention_long_rows_in_large_batches(backend, device, dim, rows, kv_heads, heads):
    """Batches that fill the chip by themselves: long rows are shared by workgroups, short ones are not, and a
    row's result does not depend on where it stands."""
    held, g = _filled(backend, device, 1, kv_heads, 36000, dim, 64, dim + rows, [36000])
    cache = Int4KvCache(*[t.expand(rows, *t.shape[1:]) for t in (held.k_codes, held.k_scales, held.v_codes, held.v_scales)])
    some = [36000, 0, 1, 8192, 8193, 16385, 32, 4096, 24577]
    lengths = [some[b] if b < len(some) else 37 * b for b in range(rows)]
    q = torch.randn((rows, heads, dim), generator=g, device=device).half()
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    out = torch.full_like(q, 5.0)
    backend.gqa_attention_int4(q, cache, out, n)
    for b in (0, 1, 2, 4, 5, 7, rows - 1):
        _check_attention(held, q[b:b + 1], out[b:b + 1], lengths[b:b + 1])
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rows)).to(device)
    mixed = torch.empty_like(q)
    backend.gqa_attention_int4(q[order].contiguous(), cache, mixed, n[order].contiguous())
    assert torch.equal(mixed, out[order])


@pytest.mark.parametrize("length", [1023, 4097, 20000])
def test_attention_split(backend, device, length):
    """Lengths that several workgroups share, beside short ones, in one call; a bound on the length."""
    lengths = [length, 5, length // 2, 0]
    cap = -(-length // 32) * 32 + 64
    cache, g = _filled(backend, device, 4, 2, cap, 128, 64, length, lengths)
    q = torch.randn((4, 10, 128), generator=g, device=device).half()
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    out = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, out, n)
    _check_attention(cache, q, out, lengths)
    again = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, again, n)
    assert torch.equal(out, again)
    again.copy_(q)
    backend.gqa_attention_int4(again, cache, again, n)          # in place
    assert torch.equal(out, again)
    short = length // 3
    backend.gqa_attention_int4(q, cache, out, n, max_length=short)
    _check_attention(cache, q, out, [min(x, short) for x in lengths])
    # lengths past the bound and the capacity count as the bound (of the rows that hold as many tokens)
    backend.gqa_attention_int4(q, cache, out, torch.where(n > short, n + 10 ** 6, n), max_length=short)
    _check_attention(cache, q, out, [min(x, short) for x in lengths])
    backend.gqa_attention_int4(q, cache, out, n * 0 - 5)
    assert torch.count_nonzero(out) == 0


def test_attention_large_scores_and_late_maximum(backend, device):
    """Scores of hundreds, the largest in the last tokens: rescales, weights that vanish."""
    lengths = [700, 90]
    cache, g = _filled(backend, device, 2, 1, 704, 64, 32, 3, lengths)
    k = torch.randn((2, 40, 1, 64), generator=g, device=device) * 12
    at = torch.tensor([660, 50], device=device, dtype=torch.int32)
    backend.kv_append_int4(cache, k, k, at)
    q = (torch.randn((2, 4, 64), generator=g, device=device) * 8).half()
    out = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, out, torch.tensor(lengths, device=device, dtype=torch.int32))
    _check_attention(cache, q, out, lengths)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
def test_attention_softmax_scales(backend, device, scale):
    """No scale (every visible token weighs the same), a negative one, one that leaves next to nothing."""
    lengths = [45, 64]
    cache, g = _filled(backend, device, 2, 2, 96, 64, 32, 6, lengths)
    q = torch.randn((2, 6, 64), generator=g, device=device).half()
    out = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, out, torch.tensor(lengths, device=device, dtype=torch.int32), scale=scale, window=40)
    _check_attention(cache, q, out, lengths, 40, scale=scale)


@pytest.mark.parametrize("scale", [2.0 ** -16, 60000.0, 2.0 ** 100, 2.0 ** -100])
def test_attention_query_range(backend, device, scale):
    """Queries near the ends of their types, with a softmax scale that brings the scores back."""
    dt = torch.float16 if 2.0 ** -20 < scale < 65504 else torch.bfloat16
    lengths = [77]
    cache, g = _filled(backend, device, 1, 2, 96, 128, 32, 4, lengths)
    q = (torch.rand((1, 4, 128), generator=g, device=device) * 2 - 1).mul_(scale).to(dt)
    out = torch.empty_like(q)
    soft = 0.1 / scale
    backend.gqa_attention_int4(q, cache, out, torch.tensor(lengths, device=device, dtype=torch.int32), scale=soft)
    _check_attention(cache, q, out, lengths, scale=float(np.float32(soft)))


def test_attention_not_finite(backend, device):
    """A query that is not finite spoils its own head alone, a poisoned group in sight every head of
    its KV head, one out of sight nothing."""
    lengths = [70, 70]
    cache, g = _filled(backend, device, 2, 2, 96, 64, 32, 8, lengths)
    q = torch.randn((2, 8, 64), generator=g, device=device).half()
    n = torch.tensor(lengths, device=device, dtype=torch.int32)
    good = torch.empty_like(q)
    backend.gqa_attention_int4(q, cache, good, n)
    bad = q.clone()
    bad[0, 1, 5], bad[0, 6, 63], bad[1, 3, 0] = float("nan"), float("inf"), float("-inf")
    out = torch.empty_like(q)
    backend.gqa_attention_int4(bad, cache, out, n)
    spoilt = torch.zeros((2, 8), dtype=torch.bool, device=device)
    spoilt[0, 1] = spoilt[0, 6] = spoilt[1, 3] = True
    assert torch.isnan(out[spoilt]).all() and torch.equal(out[~spoilt], good[~spoilt])
    x = torch.randn((2, 1, 2, 64), generator=g, device=device).half()
    x[0, 0, 1, 9] = float("nan")
    at = torch.tensor([20, 20], device=device, dtype=torch.int32)
    backend.kv_append_int4(cache, x, x, at)
    backend.gqa_attention_int4(q, cache, out, n)
    assert torch.isnan(out[0, 4:]).all() and torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()
    backend.gqa_attention_int4(q, cache, out, n, window=40, first_tokens=10)
    assert torch.isfinite(out).all()
    _check_attention(cache, q, out, lengths, 40, 10)


def test_attention_strided_rows_left_alone(backend, device):
    """Queries as parts of QKV rows, outputs inside a larger buffer, fewer rows than sequences."""
    lengths = [40, 41, 42, 43]
    cache, g = _filled(backend, device, 4, 2, 64, 64, 32, 21, lengths)
    qkv = torch.randn((3, 12 * 64 + 1), generator=g, device=device).half()
    q = qkv[:, 1:1 + 8 * 64].view(3, 8, 64)
    buf = torch.full((5, 9, 72), 7.0, device=device).half()
    n = torch.tensor(lengths[:3], device=device, dtype=torch.int32)
    backend.gqa_attention_int4(q, cache, buf[:3, :8, :64], n)
    _check_attention(cache, q, buf[:3, :8, :64], lengths[:3])
    assert torch.all(buf[3:] == 7) and torch.all(buf[:, 8] == 7) and torch.all(buf[..., 64:] == 7)
    part = cache.sequences(2, 4)
    out = torch.empty((2, 8, 64), device=device).half()
    backend.gqa_attention_int4(q[1:], part, out, torch.tensor(lengths[2:], device=device, dtype=torch.int32))
    _check_attention(part, q[1:], out, lengths[2:])
    backend.gqa_attention_int4(q[:0], cache, out[:0], n[:0])


def test_attention_past_32_bit_offsets(backend, device):
    """Heads whose codes start more than 2^31 bytes into the cache."""
    cache = Int4KvCache(torch.empty((3, 1, 32 * 1024, 8), device=device, dtype=torch.int32),
                        torch.empty((3, 1, 32 * 1024, 2, 2), device=device, dtype=torch.float16),
                        torch.empty((3, 1, 4 * 1024, 64), device=device, dtype=torch.int32),
                        torch.empty((3, 1, 4 * 1024, 2, 2, 8), device=device, dtype=torch.float16))
    far = torch.empty(3 << 28, device=device, dtype=torch.int32)              # 3 GiB
    wide = Int4KvCache(far.as_strided((3, 1, 32 * 1024, 8), (1 << 28, 1 << 28, 8, 1)), cache.k_scales,
                       far[1 << 24:].as_strided((3, 1, 4 * 1024, 64), (1 << 28, 1 << 28, 64, 1)), cache.v_scales)
    g = torch.Generator(device=device).manual_seed(2)
    n = 90
    k, v = (torch.randn((3, n, 1, 64), generator=g, device=device).half() for _ in range(2))
    starts = torch.zeros(3, device=device, dtype=torch.int32)
    backend.kv_append_int4(wide, k, v, starts)
    backend.kv_append_int4(cache, k, v, starts)
    q = torch.randn((3, 2, 64), generator=g, device=device).half()
    a, b = torch.empty_like(q), torch.empty_like(q)
    lengths = torch.full((3,), n, device=device, dtype=torch.int32)
    backend.gqa_attention_int4(q, wide, a, lengths)
    backend.gqa_attention_int4(q, cache, b, lengths)
    assert torch.equal(a, b)
    ka, va = backend.kv_read_int4(wide, torch.empty_like(k), torch.empty_like(v), starts)
    kb, vb = backend.kv_read_int4(cache, torch.empty_like(k), torch.empty_like(v), starts)
    assert torch.equal(ka, kb) and torch.equal(va, vb)


def test_attention_and_read_over_a_shared_sequence(backend, device):
    """One sequence seen by every row (stride 0): read and attended to as copies of it, never written."""
    held, g = _filled(backend, device, 1, 2, 288, 128, 64, 77, [288])
    arrays = (held.k_codes, held.k_scales, held.v_codes, held.v_scales)
    shared = Int4KvCache(*[t.expand(5, *t.shape[1:]) for t in arrays])
    copies = Int4KvCache(*[t.repeat(5, *[1] * (t.ndim - 1)) for t in arrays])
    q = torch.randn((5, 8, 128), generator=g, device=device).half()
    n = torch.tensor([288, 1, 100, 0, 37], device=device, dtype=torch.int32)
    outs = [torch.empty_like(q) for _ in range(2)]
    for cache, out in zip((shared, copies), outs):
        backend.gqa_attention_int4(q, cache, out, n)
    assert torch.equal(*outs)
    starts = torch.tensor([0, 8, 100, 287, 5], device=device, dtype=torch.int32)
    rows = [[torch.full((5, 9, 2, 128), 3.0, device=device).half() for _ in range(2)] for _ in range(2)]
    for cache, out in zip((shared, copies), rows):
        backend.kv_read_int4(cache, *out, starts)
    assert all(torch.equal(a, b) for a, b in zip(*rows))
    with pytest.raises(ValueError, match="share"):
        backend.kv_append_int4(shared, rows[0][0][:, 0], rows[0][1][:, 0], starts)
