"""YaRN frequencies against their definition, one by one: rounded and unrounded ends of the ramp."""

from __future__ import annotations

import math

import numpy as np
import pytest

from thintensor_amd.rotary import rotary_frequencies


def _yarn(dim, theta, factor, original, fast, slow, truncate):
    end = [dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (fast, slow)]
    if truncate:
        end = [math.floor(end[0]), math.ceil(end[1])]
    end = [max(end[0], 0), min(end[1], dim - 1)]
    out = []
    for i in range(dim // 2):
        f = theta ** (-2 * i / dim)
        if end[1] > end[0]:
            ramp = min(max((i - end[0]) / (end[1] - end[0]), 0.0), 1.0)
        else:
            ramp = float(i > end[0])
        out.append(f * (1 - ramp) + f / factor * ramp)
    return out


@pytest.mark.parametrize("truncate", [True, False])
@pytest.mark.parametrize("dim,theta,factor,original,fast,slow", [
    (64, 150000.0, 32.0, 4096, 32.0, 1.0), (128, 10000.0, 4.0, 4096, 32.0, 1.0), (96, 500000.0, 16.0, 8192, 16.0, 2.0),
    (64, 10000.0, 8.0, 100, 32.0, 1.0), (32, 100.0, 2.0, 100000, 4.0, 1.0)])
def test_yarn_frequencies(dim, theta, factor, original, fast, slow, truncate):
    got, amplitude = rotary_frequencies(dim, theta, scaling="yarn", factor=factor, original_positions=original, beta_fast=fast,
                                        beta_slow=slow, truncate=truncate, device="cpu")
    np.testing.assert_allclose(got.numpy(), _yarn(dim, theta, factor, original, fast, slow, truncate), rtol=1e-12)
    assert math.isclose(amplitude, 0.1 * math.log(factor) + 1.0)


def test_yarn_ends_of_the_published_gpt_oss_settings():
    """Unrounded, the ramp runs from index 8.09 to 17.40; the frequencies between differ from the rounded ones."""
    settings = dict(scaling="yarn", factor=32.0, original_positions=4096, device="cpu")
    rounded, _ = rotary_frequencies(64, 150000.0, **settings)
    exact, _ = rotary_frequencies(64, 150000.0, truncate=False, **settings)
    base, _ = rotary_frequencies(64, 150000.0, device="cpu")
    keep = ((exact / base).numpy() - 1 / 32) / (1 - 1 / 32)
    assert np.all(keep[:9] == 1.0) and np.all(np.abs(keep[18:]) < 1e-12)
    np.testing.assert_allclose(keep[9:18], 1 - (np.arange(9, 18) - 8.0928) / (17.3980 - 8.0928), atol=2e-4)
    assert np.all(rounded.numpy()[9:18] != exact.numpy()[9:18]) and np.array_equal(rounded.numpy()[:9], exact.numpy()[:9])
