"""rotary_rows against its definition in float64.

Error of an output before its rounding: the reduced turn is rounded to binary32 (at most 2^-26 of a
turn, 2^-23.3 radians), sine and cosine, the amplitude and the two products and their sum add at most
five roundings of 2^-24: below 2^-21 amplitude (|a| + |b|).  The store adds half a step of its type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref
from thintensor_amd.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _check(got, x, positions, freq, interleaved, amplitude, dtype):
    want = step_ref.rotary(x, positions, freq, interleaved, amplitude)
    r = 2 * len(freq)
    size = np.abs(x)
    pair = size.copy()
    if interleaved:
        pair[..., :r] = (size[..., :r].reshape(*x.shape[:-1], -1, 2).sum(-1)).repeat(2, -1)
    else:
        pair[..., :r] = np.concatenate([size[..., :r // 2] + size[..., r // 2:r]] * 2, -1)
    err = np.abs(got.double().cpu().numpy() - want)
    info = torch.finfo(dtype)
    bound = 2.0 ** -21 * amplitude * pair + info.eps / 2 * np.abs(want) * (1 + 2.0 ** -20) + info.tiny * info.eps
    assert np.all(err <= bound), float((err - bound).max())
    assert np.array_equal(got.double().cpu().numpy()[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [
    (1, 32, 8, 64, 64), (3, 4, 1, 128, 32), (5, 3, 3, 80, 20), (2, 5, 0, 256, 256), (17, 2, 2, 6, 2), (1, 1, 1, 1024, 96)])
def test_rotary(backend, device, dtype, interleaved, tokens, heads, kv_heads, dim, rotary):
    g = torch.Generator(device=device).manual_seed(tokens * 1000 + dim + interleaved)
    dt = _DT[dtype]
    q = torch.randn((tokens, heads, dim), generator=g, device=device).to(dt)
    k = torch.randn((tokens, kv_heads, dim), generator=g, device=device).to(dt) if kv_heads else None
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device=device, dtype=torch.int32)
    freq, amp = rotary_frequencies(rotary, 150000.0, scaling="linear", factor=2.0, device=device)
    amp = 1.25
    qo, ko = torch.empty_like(q), torch.empty_like(k) if k is not None else None
    backend.rotary_rows(q, k, pos, freq, qo, ko, interleaved=interleaved, amplitude=amp)
    p, f = pos.cpu().numpy(), freq.cpu().numpy()
    _check(qo, q.double().cpu().numpy(), p, f, interleaved, amp, dt)
    if k is not None:
        _check(ko, k.double().cpu().numpy(), p, f, interleaved, amp, dt)
    q2, k2 = q.clone(), k.clone() if k is not None else None
    backend.rotary_rows(q2, k2, pos.long(), freq, interleaved=interleaved, amplitude=amp)     # in place, int64
    assert torch.equal(q2, qo) and (k is None or torch.equal(k2, ko))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_strides_and_far_positions(backend, device, interleaved):
    """A QKV row's parts as strided views, a misaligned one too; positions past 2^31 and negative ones."""
    g = torch.Generator(device=device).manual_seed(7)
    tokens, heads, kv, dim = 9, 4, 2, 64
    qkv = torch.randn((tokens, (heads + 2 * kv) * dim + 1), generator=g, device=device).half()
    pos = torch.tensor([0, 1, -1, 131071, 2 ** 31 + 5, -(2 ** 33), 2 ** 40 + 3, 7, 8], device=device)
    freq, _ = rotary_frequencies(32, 10000.0, device=device)
    for shift in (0, 1):
        q = qkv[:, shift:shift + heads * dim].view(tokens, heads, dim)
        k = qkv[:, shift + heads * dim:shift + (heads + kv) * dim].view(tokens, kv, dim)
        before = qkv.clone()
        qo = torch.zeros((tokens, kv + heads, dim + 8), device=device).half()
        backend.rotary_rows(q, k, pos, freq, qo[:, :heads, :dim], qo[:, heads:, :dim], interleaved=interleaved)
        assert torch.equal(qkv, before) and torch.count_nonzero(qo[..., dim:]) == 0
        # past 2^31 binary64 itself leaves 2^-52 of the angle: the first frequency's, 1 radian a position
        near = pos.abs() < 2 ** 32
        for x, o in ((q, qo[:, :heads, :dim]), (k, qo[:, heads:, :dim])):
            _check(o[near], x[near].double().cpu().numpy(), pos[near].cpu().numpy(), freq.cpu().numpy(), interleaved, 1.0,
                   torch.float16)
            assert torch.isfinite(o.float()).all()
        backend.rotary_rows(q, k, pos, freq, interleaved=interleaved)
        assert torch.equal(q, qo[:, :heads, :dim]) and torch.equal(k, qo[:, heads:, :dim])
        assert torch.equal(qkv[:, shift + (heads + kv) * dim:], before[:, shift + (heads + kv) * dim:])
        qkv.copy_(before)


def test_rotary_no_tokens(backend, device):
    q = torch.empty((0, 4, 64), device=device).half()
    freq, _ = rotary_frequencies(64, device=device)
    assert backend.rotary_rows(q, None, torch.empty(0, device=device, dtype=torch.int32), freq)[0].shape == (0, 4, 64)
