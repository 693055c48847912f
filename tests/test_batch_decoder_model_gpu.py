"""The batch decoder's steps against the model in float64: embeddings, norms, projections, the rotation to
each request's position, what the caches take, attention over what they hold, residuals, the MLP, logits.

Every operator rounds its output to fp16, 2^-11 of an element at most, and about twenty-five of them lie on
the way to a logit.  Independent, they make 5 x 2^-11 of a row's norm; a norm, a product of two roundings
or a softmax over scores of a few units takes such an error up to fourfold: 2^-6.7, below the 1e-2 of a
row's norm that is allowed.  The mistakes that the last test plants in the restatement are at least ten
times as far away."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.cpu_path import dequant_int4
from tests import step_ref
from tests.test_kv_int4_gpu import _held
from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.decode import DenseBatchDecoder
from thintensor_amd.rotary import rotary_frequencies
from thintensor_amd.synth import DenseShape, make_dense

pytestmark = pytest.mark.gpu

_SHAPE = DenseShape(name="wiring", layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, intermediate=1024, vocab=1000,
                    prior_tokens=40, max_new_tokens=8)
_ALLOWED = 1e-2


@pytest.fixture(scope="module")
def model(device):
    w = make_dense(_SHAPE, device=device, seed=11, centered_codes=True)
    g = torch.Generator(device=device).manual_seed(12)
    for t in [w.final_norm] + [t for L in w.layers for t in (L.ln1, L.ln2)]:
        t.copy_(1 + 0.3 * torch.randn(t.shape, generator=g, device=device))
    return w


def _plain(model):
    """The model's weights in float64 on the host."""
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    dense = lambda p: dequant_int4(p[0].cpu(), p[1].cpu(), _SHAPE.group).double().numpy()  # noqa: E731
    layers = [{n: dense(getattr(L, n)) for n in ("q", "k", "v", "o", "gate", "up", "down")} | {"ln1": f(L.ln1), "ln2": f(L.ln2)}
              for L in model.layers]
    return {"embed": f(model.embed), "head": f(model.lm_head), "norm": f(model.final_norm), "layers": layers}


def _rms(x, w):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + _SHAPE.eps) * w


def _model(w, tokens, positions, freq, amplitude, held, window, first, mistake=None):
    """Logits [batch, vocab] and each layer's rotated k and v [batch, kv_heads, dim]; held[layer][request]:
    K and V [kv_heads, tokens, dim] up to and with the new token."""
    s, B = _SHAPE, len(tokens)
    pos = np.asarray(positions) + (1 if mistake == "position" else 0)
    if mistake == "shared position":
        pos = np.full(B, positions[0])
    x, made = w["embed"][np.asarray(tokens)], []
    for li, L in enumerate(w["layers"]):
        n = _rms(x, L["ln1"])
        q, k = ((n @ L[c].T).reshape(B, h, s.head_dim) for c, h in (("q", s.heads), ("k", s.kv_heads)))
        q, k = (step_ref.rotary(t, pos, freq, mistake == "pairs", amplitude) for t in (q, k))
        made.append((k, (n @ L["v"].T).reshape(B, s.kv_heads, s.head_dim)))
        out = [step_ref.attention(q[b], *held[li][b], positions[b] + (0 if mistake == "length" else 1), window,
                                  first)[0].reshape(-1) for b in range(B)]
        y = x + np.stack(out) @ L["o"].T
        n = _rms(y, L["ln1" if mistake == "norm" else "ln2"])
        g = n @ L["gate"].T
        x = (x if mistake == "residual" else y) + (g / (1 + np.exp(-g)) * (n @ L["up"].T)) @ L["down"].T
    return _rms(x, w["norm"]) @ w["head"].T, made


def _decoder(device, model, lengths, window, first, rotary):
    s = _SHAPE
    be = HipDecodeBackend(device, torch.float16, s.hidden, s.q_dim, s.kv_dim, s.intermediate)
    dec = DenseBatchDecoder(be, model, len(lengths), 96, window=window, first_tokens=first, rotary=rotary)
    g = torch.Generator(device=device).manual_seed(13)
    for li in range(s.layers):
        k, v = (torch.randn((len(lengths), max(lengths) + 1, s.kv_heads, s.head_dim), generator=g, device=device).half() for _ in range(2))
        dec.append(li, k, v, torch.zeros(len(lengths), device=device, dtype=torch.int32), torch.tensor(lengths, device=device, dtype=torch.int32))
    return dec




def _all_held(dec, positions):
    return [[[step_ref.dequantize(c[:, :p + 1], st[:, :p + 1], m[:, :p + 1]) for c, st, m in _held(cache, b)] for b, p in enumerate(positions)]
            for cache in dec.caches]


def _off(got, want):
    return float((np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)).max())


@pytest.mark.parametrize("lengths", [[40], [0, 33], [40, 1, 33, 0, 64]])
@pytest.mark.parametrize("window,first,scaling", [(0, 0, None), (16, 3, None), (0, 0, "yarn")])
def test_steps_against_the_model(device, model, lengths, window, first, scaling):
    """Batches of both forms of the GEMMs, three steps each."""
    w = _plain(model)
    rotary = rotary_frequencies(64, 10000.0, scaling=scaling, factor=4.0 if scaling else 1.0, original_positions=32, device=device)
    dec = _decoder(device, model, lengths, window, first, rotary)
    dec.set_sampling(1.0, 20)
    dec.uniforms.copy_(torch.linspace(0.1, 0.9, len(lengths)))
    dec.prime([7 + 90 * b for b in range(len(lengths))], lengths)
    for _ in range(3):
        tokens, positions = dec.tokens.tolist(), dec.positions.tolist()
        dec.step()
        held = _all_held(dec, positions)
        want, made = _model(w, tokens, positions, rotary[0].cpu().numpy(), rotary[1], held, window, first)
        got = dec.logits.double().cpu().numpy()
        assert _off(got, want) <= _ALLOWED, _off(got, want)
        for li, cache in enumerate(dec.caches):
            for b, p in enumerate(positions):
                for x, (codes, st, m), kept in zip(made[li], _held(cache, b), held[li][b]):
                    # half a step of its group, and what the operators before it may be off by
                    room = np.repeat(st[:, p], cache.group_size, -1) * 0.5 + _ALLOWED * np.linalg.norm(x[b], axis=-1, keepdims=True)
                    assert np.all(np.abs(kept[:, p] - x[b]) <= room), (li, b)


def test_planted_mistakes_are_seen(device, model):
    lengths = [40, 1, 33, 10, 64]
    w, rotary = _plain(model), rotary_frequencies(64, 10000.0, device=device)
    dec = _decoder(device, model, lengths, 0, 0, rotary)
    dec.prime([7 + 90 * b for b in range(5)], lengths)
    tokens = dec.tokens.tolist()
    dec.step()
    held, got = _all_held(dec, lengths), dec.logits.double().cpu().numpy()
    freq = rotary[0].cpu().numpy()
    assert _off(got, _model(w, tokens, lengths, freq, 1.0, held, 0, 0)[0]) <= _ALLOWED
    for mistake in ("position", "shared position", "pairs", "length", "norm", "residual"):
        assert _off(got, _model(w, tokens, lengths, freq, 1.0, held, 0, 0, mistake)[0]) > 10 * _ALLOWED, mistake
