"""What the batch decoder refuses before anything is launched."""

from __future__ import annotations

import pytest
import torch

from thintensor_amd import _lib
from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.decode import DenseBatchDecoder
from thintensor_amd.synth import DenseShape, make_dense

_SHAPE = DenseShape(name="refuse", layers=1, hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=256, vocab=300,
                    prior_tokens=4, max_new_tokens=2)


@pytest.fixture(scope="module")
def decoder():
    if not _lib.library_path().exists():
        pytest.skip("kernel library not built (run __graft_entry__.build())")
    cpu = torch.device("cpu")
    be = HipDecodeBackend(cpu, torch.float16, _SHAPE.hidden, _SHAPE.q_dim, _SHAPE.kv_dim, _SHAPE.intermediate)
    return DenseBatchDecoder(be, make_dense(_SHAPE, device=cpu, seed=1), 2, 32)


def test_start_tokens_outside_the_vocabulary(decoder):
    """The embedding leaves a row as it was for such an id, so the step would start from another request's."""
    decoder.prime([0, _SHAPE.vocab - 1], [0, 31])
    held = decoder.tokens.tolist(), decoder.positions.tolist()
    for tokens in ([_SHAPE.vocab, 0], [0, -1], [1 << 40, 3]):
        with pytest.raises(ValueError, match="vocabulary"):
            decoder.prime(tokens, [1, 1])
        with pytest.raises(ValueError, match="vocabulary"):
            decoder.generate(tokens, [1, 1], torch.zeros((1, 2)), use_graph=False)
    assert (decoder.tokens.tolist(), decoder.positions.tolist()) == held
