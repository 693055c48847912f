"""Frequencies for ``HipDecodeBackend.rotary_rows``, formed once on the host in binary64.

Frequency i of a rotation of ``rotary_dim`` dims is theta ** (-2 i / rotary_dim) radians per
position.  For contexts longer than a model was trained on, the published scalings are offered:

* ``"linear"``: every frequency divided by ``factor``;
* ``"ntk"``: theta times factor ** (rotary_dim / (rotary_dim - 2)), which divides the lowest
  frequency by the factor and leaves the highest;
* ``"yarn"``: frequencies that turn more than ``beta_fast`` times over ``original_positions`` are kept,
  those that turn less than ``beta_slow`` times are divided by the factor, with a linear ramp over the
  index between, whose ends are rounded outwards to whole indices unless ``truncate`` is false (as in
  gpt-oss's settings); vectors grow by 0.1 ln(factor) + 1;
* ``"bands"``: by wavelength: kept below original_positions / ``high_freq_factor``, divided by the
  factor above original_positions / ``low_freq_factor``, blended linearly in original_positions /
  wavelength between.
"""

from __future__ import annotations

import math

import torch


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       original_positions: int = 8192, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       truncate: bool = True, low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                       device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim / 2] on ``device``, amplitude)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not (0 < theta < math.inf and 1 <= factor < math.inf):
        raise ValueError("rotary theta must be positive and the factor at least 1, both finite")
    half = rotary_dim // 2
    index = torch.arange(half, dtype=torch.float64)
    freq = theta ** (-2.0 * index / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs at least two frequencies")
        freq = (theta * factor ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * index / rotary_dim)
    elif scaling == "yarn":
        if theta <= 1 or original_positions < 1 or not 0 < beta_slow < beta_fast:
            raise ValueError("yarn scaling needs theta above 1, original positions and 0 < beta_slow < beta_fast")

        # index at which a frequency turns `turns` times over the original positions
        def at(turns: float) -> float:
            return rotary_dim * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low, high = at(beta_fast), at(beta_slow)
        if truncate:
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        ramp = ((index - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling == "bands":
        if not 0 < low_freq_factor < high_freq_factor:
            raise ValueError("band scaling needs 0 < low_freq_factor < high_freq_factor")
        turns = original_positions * freq / (2.0 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    elif scaling is not None:
        raise ValueError(f"unknown rotary scaling {scaling!r}")
    return freq.to(device), amplitude
