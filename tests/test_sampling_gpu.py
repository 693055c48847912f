"""sample_rows against its definition in float64: tokens equal; a share is rounded to binary32 (2^-24)
after sums in units of 2^-43 of the largest weight, half a unit off for each kept token."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _check(backend, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows, vocab = logits.shape
    dev = logits.device
    as_t = lambda x, dt: None if x is None else torch.as_tensor(x, dtype=dt, device=dev).expand(rows).contiguous()  # noqa: E731
    u, t, k, p, m = (as_t(u, torch.float32), as_t(temperature, torch.float32), as_t(top_k, torch.int32),
                     as_t(top_p, torch.float32), as_t(min_p, torch.float32))
    tokens = torch.full((rows,), -7, device=dev, dtype=torch.int64)
    probs = torch.full((rows,), -7.0, device=dev)
    backend.sample_rows(logits, u, tokens, temperature=t, top_k=k, top_p=p, min_p=m, probs=probs)
    x = logits.double().cpu().numpy()
    at = lambda v, i, d: d if v is None else v[i].item()  # noqa: E731
    for i in range(rows):
        token, share = step_ref.sample(x[i], u[i].item(), at(t, i, 1.0), at(k, i, 0), at(p, i, 1.0), at(m, i, 0.0))
        assert tokens[i].item() == token, (i, tokens[i].item(), token, share, probs[i].item())
        assert abs(probs[i].item() - share) <= share * (2.0 ** -23 + vocab * 2.0 ** -43), (i, probs[i].item(), share)
    return tokens, probs


def _logits(device, rows, vocab, dtype, seed, std=2.5):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device=device) * std
    return x.to(_DT[dtype]), torch.rand(rows, generator=g, device=device), g


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 1000, 1025, 8191, 32000, 128256])
def test_sample_settings(backend, device, dtype, vocab):
    rows = 24
    x, u, g = _logits(device, rows, vocab, dtype, vocab)
    i = torch.arange(rows)
    temperature = torch.tensor([0.7, 1.0, 1.5, 0.3, 5.0, 0.0])[i % 6]
    top_k = torch.tensor([0, 1, 2, 50, 1000, vocab, vocab + 5, -3])[i % 8]
    top_p = torch.tensor([1.0, 0.9, 0.5, 0.05, 0.0, 2.0, 0.999])[i % 7]
    min_p = torch.tensor([0.0, 0.02, 0.5, 1.0, 1.5])[i % 5]
    _check(backend, x, u)
    _check(backend, x, u, temperature)
    _check(backend, x, u, 0.9, top_k)
    _check(backend, x, u, 1.1, None, top_p)
    _check(backend, x, u, 1.3, None, None, min_p)
    _check(backend, x, u, temperature, top_k, top_p, min_p)


def test_sample_uniforms_at_their_ends(backend, device):
    x, _, _ = _logits(device, 8, 5000, "f16", 3)
    u = [0.0, 1.0, 1.5, -1.0, float("nan"), 1 - 2.0 ** -24, 2.0 ** -149, 0.5]
    _check(backend, x, u)
    _check(backend, x, u, 0.5, 100, 0.9)


def test_sample_cumulative_walk(backend, device):
    """Every u on a grid: the tokens are those of the inverse distribution, and their shares are equal
    to how often they come."""
    w = torch.tensor([1.0, 4.0, 2.0, 4.0, 5.0], device=device)
    n = 4096
    x = w.log()[None].expand(n, 5)
    u = (torch.arange(n, device=device) + 0.5) / n
    tokens, probs = _check(backend, x.contiguous(), u)
    assert torch.equal(torch.bincount(tokens, minlength=5).float(), w / 16 * n)
    assert torch.all(tokens[: 5 * n // 16] == 4) and torch.all(tokens[-n // 16:] == 0)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_sample_masks(backend, device, dtype):
    """Rows masked by -inf, by the type's lowest value and by NaN; rows with one token or none left;
    +inf; -0 beside +0."""
    x, u, g = _logits(device, 12, 3001, dtype, 17)
    keep = torch.rand(x.shape, generator=g, device=device) < 0.01
    low = torch.finfo(x.dtype).min
    x[0:2] = x[0:2].masked_fill(~keep[0:2], float("-inf"))
    x[2:4] = x[2:4].masked_fill(~keep[2:4], low)
    x[4:6] = x[4:6].masked_fill(~keep[4:6], float("nan"))
    x[6] = float("-inf")
    x[7] = float("nan")
    x[8] = float("-inf")
    x[8, 2999] = -3.0
    x[9] = low
    x[10, 5], x[10, 77], x[10, 78] = float("inf"), float("inf"), float("nan")
    x[11] = -1.0
    x[11, 10::20], x[11, 5::20] = -0.0, 0.0
    for temperature in (None, 0.6, 0.0, 3.0):
        for top_k, top_p, min_p in ((None, None, None), (40, 0.8, 0.01), (2000, None, None), (None, 0.3, None)):
            tokens, probs = _check(backend, x, u, temperature, top_k, top_p, min_p)
            assert tokens[6].item() == tokens[7].item() == -1 and probs[6].item() == 0.0
            assert tokens[8].item() == 2999


@pytest.mark.parametrize("vocab", [5000, 40000])
def test_sample_many_equal_logits(backend, device, vocab):
    """More candidates than are sorted at once: a flat row, two levels, a few values only."""
    g = torch.Generator(device=device).manual_seed(vocab)
    x = torch.zeros((6, vocab), device=device)
    x[1, ::3] = 1.0
    x[2] = torch.randint(0, 4, (vocab,), generator=g, device=device).float()
    x[3, vocab // 2:] = -40.0
    x[4] = -65504.0
    x[5] = torch.randint(0, 2, (vocab,), generator=g, device=device).float() * 100.0
    u = torch.rand(6, generator=g, device=device)
    for k, p, m in ((None, None, None), (vocab // 2 + 1, None, None), (None, 0.37, None), (None, None, 0.9),
                    (vocab - 7, 0.61, 0.2)):
        for t in (1.0, 0.7):
            _check(backend, x.half(), u, t, k, p, m)


def test_sample_temperatures_far_from_one(backend, device):
    x, u, _ = _logits(device, 7, 20011, "f32", 23)
    _check(backend, x, u, torch.tensor([1e-30, 1e-3, 100.0, 1e6, 1e30, float("nan"), float("inf")]), None, 0.95)
    _check(backend, x * 1e30, u, torch.tensor([1.0, 1e28, 1e30, 1e35, 1e-30, -1.0, 3e38]), 500)
    _check(backend, x * 1e-30, u, torch.tensor([1.0, 1e-28, 1e-30, 1e-32, 1e30, 0.0, 1e-38]), 500, 0.9)


@pytest.mark.parametrize("vocab", [30, 3126, 20000])
@pytest.mark.parametrize("temperature", [1e3, 1e30])
def test_sample_min_p_at_high_temperatures(backend, device, vocab, temperature):
    """Weights that are all 1, or nearly: a logit passes min-p by what its weight rounds to, however many
    bins of the row that is."""
    x, u, _ = _logits(device, 12, vocab, "f32", vocab)
    top_k = torch.tensor([0, 7, vocab - 1])[torch.arange(12) % 3]
    for min_p in (1.0, 1.0 - 2.0 ** -24, 0.999, 0.5, 2.0):
        _check(backend, x, u, temperature, None, None, min_p)
        _check(backend, x, u, temperature, top_k, 0.7, min_p)


@pytest.mark.parametrize("stride", [0, 1, 3, 8])
def test_sample_row_strides(backend, device, stride):
    """Rows inside a wider buffer, from an odd first element; many rows at once."""
    x, u, g = _logits(device, 130, 1024 + stride, "bf16", 31)
    view = x[:, stride:] if stride else x
    _check(backend, view, u, 0.8, 20, 0.95)
    one = x[0, stride:][None].expand(130, 1024)         # one row for all requests
    _check(backend, one, u, 0.8, 20, 0.95)


def test_sample_distribution(backend, device):
    """Frequencies over many uniforms: within five standard deviations of the kept shares."""
    x, _, g = _logits(device, 1, 300, "f32", 41, 1.5)
    n = 20000
    u = torch.rand(n, generator=g, device=device)
    tokens = torch.empty(n, device=device, dtype=torch.int64)
    probs = torch.empty(n, device=device)
    top_p = torch.full((n,), 0.8, device=device)
    backend.sample_rows(x.expand(n, 300), u, tokens, top_p=top_p, probs=probs)
    share = torch.zeros(300, device=device)
    share[tokens] = probs
    assert abs(share.sum().item() - 1.0) < 2e-2          # nearly every kept token came up
    seen = torch.bincount(tokens, minlength=300).float()
    sd = (n * share * (1 - share)).sqrt() + 1e-9
    assert torch.all((seen - n * share).abs() <= 5 * sd + 1)


def test_sample_without_shares_and_no_rows(backend, device):
    x, u, _ = _logits(device, 3, 100, "f16", 2)
    a, b = (torch.empty(3, device=device, dtype=torch.int64) for _ in range(2))
    backend.sample_rows(x, u, a)
    backend.sample_rows(x, u, b, probs=torch.empty(3, device=device))
    assert torch.equal(a, b)
    backend.sample_rows(x[:0], u[:0], a[:0])
