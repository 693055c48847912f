"""The batch decoder's requests that have no token left."""

from __future__ import annotations

import pytest
import torch

from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.decode import DenseBatchDecoder
from thintensor_amd.synth import DenseShape, make_dense

pytestmark = pytest.mark.gpu

_SHAPE = DenseShape(name="batch", layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, intermediate=1024, vocab=4096,
                    prior_tokens=40, max_new_tokens=8)


@pytest.fixture(scope="module")
def model(device):
    return make_dense(_SHAPE, device=device, seed=3, centered_codes=True)


def _decoder(device, model, batch, capacity=96, **kw):
    s = _SHAPE
    be = HipDecodeBackend(device, torch.float16, s.hidden, s.q_dim, s.kv_dim, s.intermediate)
    return DenseBatchDecoder(be, model, batch, capacity, **kw)


def _stored(dec, b):
    return [t[b].clone() for c in dec.caches for t in (c.k_codes, c.v_codes, c.k_scales.view(torch.int16), c.v_scales.view(torch.int16))]


@pytest.mark.parametrize("batch", [1, 3, 6])           # both forms of the batched GEMMs
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_token_minus_one_stays(device, model, batch, use_graph, temperature):
    """Token -1 reads nothing that an earlier step left, whatever that is, and gives -1 again; the other
    requests' tokens and caches are what they are without it."""
    last, runs = batch - 1, []
    starts, positions = [5 + 100 * b for b in range(batch)], [3 * b for b in range(batch)]
    for junk in (None, 0.0, 1.0, float("inf")):
        dec = _decoder(device, model, batch)
        dec.set_sampling(temperature)
        dec.uniforms.fill_(0.4)
        if use_graph:
            dec.capture()
        dec.prime(starts, positions)
        tokens = []
        for step in range(4):
            if junk is not None and step == 1:
                dec.tokens[last] = -1
                dec.embedded.fill_(junk)
            dec.graph.replay() if use_graph else dec.step()
            tokens.append(dec.tokens.tolist())
        if junk is not None:
            assert [t[last] for t in tokens[1:]] == [-1, -1, -1], junk
            assert dec.probs[last].item() == 0.0
        runs.append(([t[:last] for t in tokens], [_stored(dec, b) for b in range(last)]))
        # primed again, it is a request like any other
        dec.prime(starts, positions)
        dec.graph.replay() if use_graph else dec.step()
        assert dec.tokens.tolist() == tokens[0]
    assert all(min(t) >= 0 for t in runs[0][0] if t)
    for tokens, stored in runs[1:]:
        assert tokens == runs[0][0]
        for a, b in zip(stored, runs[0][1]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
