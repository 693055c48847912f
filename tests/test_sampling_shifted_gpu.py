"""sample_rows on rows of 16-bit logits far from zero: their spacing puts thousands of equal logits at a
border, more than are sorted at once.  Tokens are those of the float64 definition; a share as in
test_sampling_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref

pytestmark = pytest.mark.gpu

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _equal_at_borders(x, temperature, top_p, token):
    """How many logits of the row equal the last one that top-p keeps, or the token's."""
    order = np.sort(x[np.isfinite(x)])[::-1]
    cum = np.cumsum(np.exp((order - order[0]) / temperature))
    last = order[np.searchsorted(cum, top_p * cum[-1])]
    return int(np.count_nonzero((x == last) | (x == x[token])))


@pytest.mark.parametrize("dtype,mean,vocab", [("bf16", 20.0, 201088), ("bf16", -20.0, 201088), ("bf16", 20.0, 128256), ("bf16", -24.0, 40001),
                                              ("bf16", 100.0, 65537), ("f16", 20.0, 201088), ("f16", 200.0, 128256)])
def test_shifted_logits(backend, device, dtype, mean, vocab):
    rows = 6
    g = torch.Generator(device=device).manual_seed(vocab + int(mean))
    x = (torch.randn((rows, vocab), generator=g, device=device) * 2 + mean).to(_DT[dtype])
    if vocab % 2 == 0:
        x[1] = x[1].masked_fill(torch.rand(vocab, generator=g, device=device) < 0.4, float("-inf"))
    held = x.double().cpu().numpy()
    u = torch.tensor([0.0, 0.3, 0.55, 0.8, 0.95, 1 - 2.0 ** -24], device=device)
    i = torch.arange(rows, device=device)
    many = 0
    for t, k, p, m in ((1.0, 0, 0.95, 0.0), (1.2, 0, 0.95, 0.0), (2.0, 0, 0.9, 0.0), (1.0, vocab // 20, 1.0, 0.0), (1.5, vocab // 7, 0.8, 0.0),
                       (1.0, 0, 1.0, 0.02), (2.0, vocab // 3, 0.97, 0.05), (0.7, 0, 1.0, 0.0), (4.0, 0, 0.5, 0.0)):
        settings = dict(temperature=torch.full((rows,), t, device=device), top_k=torch.full((rows,), k, device=device, dtype=torch.int32),
                        top_p=torch.full((rows,), p, device=device), min_p=torch.full((rows,), m, device=device))
        settings["temperature"][i == 4] *= 1.3                       # rows of one call differ
        tokens, probs = torch.full((rows,), -7, device=device, dtype=torch.int64), torch.full((rows,), -7.0, device=device)
        backend.sample_rows(x, u, tokens, probs=probs, **settings)
        for b in range(rows):
            args = [settings[n][b].item() for n in ("temperature", "top_k", "top_p", "min_p")]
            token, share = step_ref.sample(held[b], u[b].item(), *args)
            assert tokens[b].item() == token, (t, k, p, m, b, tokens[b].item(), token)
            assert abs(probs[b].item() - share) <= share * (2.0 ** -23 + vocab * 2.0 ** -43), (t, k, p, m, b)
            if k == 0 and p < 1:
                many += _equal_at_borders(held[b], args[0], args[2], token) > 4096
    assert many > 0 or vocab < 200000 or dtype == "f16"              # rows that are searched, not sorted
