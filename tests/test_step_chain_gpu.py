"""The operators of a decode step around its weights as they run together: a batch decoder, captured
and replayed graphs, side streams."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import step_ref
from tests.test_kv_int4_gpu import _check_attention, _held
from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.decode import DenseBatchDecoder
from thintensor_amd.kv_cache import Int4KvCache
from thintensor_amd.rotary import rotary_frequencies
from thintensor_amd.synth import DenseShape, make_dense

pytestmark = pytest.mark.gpu

_SHAPE = DenseShape(name="chain", layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, intermediate=1024, vocab=4096,
                    prior_tokens=40, max_new_tokens=8)


@pytest.fixture(scope="module")
def model(device):
    return make_dense(_SHAPE, device=device, seed=3, centered_codes=True)


def _decoder(device, model, batch, capacity=96, **kw):
    s = _SHAPE
    be = HipDecodeBackend(device, torch.float16, s.hidden, s.q_dim, s.kv_dim, s.intermediate)
    return DenseBatchDecoder(be, model, batch, capacity, **kw)


def _prior(dec, order, lengths, seed=0):
    """Tokens that request order[b] holds, the same whichever row it is in."""
    for li in range(len(dec.caches)):
        k, v = [], []
        for r in order:
            g = torch.Generator(device=dec.device).manual_seed(1000 * seed + 10 * r + li)
            k.append(torch.randn((max(lengths), _SHAPE.kv_heads, _SHAPE.head_dim), generator=g, device=dec.device).half())
            v.append(torch.randn((max(lengths), _SHAPE.kv_heads, _SHAPE.head_dim), generator=g, device=dec.device).half())
        dec.append(li, torch.stack(k), torch.stack(v), torch.zeros(len(order), device=dec.device, dtype=torch.int32),
                   torch.tensor([lengths[r] for r in order], device=dec.device, dtype=torch.int32))


def _run(device, model, order, lengths, uniforms, use_graph, **kw):
    dec = _decoder(device, model, len(order), **kw)
    pick = lambda x: [x[r] for r in order]  # noqa: E731
    dec.set_sampling(pick([0.0, 0.8, 1.3, 0.7, 1.0]), pick([0, 50, 0, 7, 0]), pick([1.0, 0.9, 0.6, 1.0, 1.0]),
                     pick([0.0, 0.0, 0.0, 0.0, 0.05]))
    _prior(dec, order, lengths)
    return dec, dec.generate(pick([5, 17, 900, 4000, 33]), pick(lengths), uniforms[:, order].contiguous(), use_graph)


@pytest.mark.parametrize("kw", [{}, {"window": 16, "first_tokens": 3}, {"group_size": 64}])
def test_batch_decoder(device, model, kw):
    """A graph gives what eager calls give, requests do not depend on their row, and the last step's
    buffers are what the definitions make of them."""
    lengths = [40, 1, 33, 0, 64]
    g = torch.Generator(device=device).manual_seed(1)
    uniforms = torch.rand((7, 5), generator=g, device=device)
    dec, eager = _run(device, model, [0, 1, 2, 3, 4], lengths, uniforms, False, **kw)
    _, graph = _run(device, model, [0, 1, 2, 3, 4], lengths, uniforms, True, **kw)
    assert graph == eager
    mixed = [3, 0, 4, 1, 2]
    _, other = _run(device, model, mixed, lengths, uniforms, True, **kw)
    assert [other[mixed.index(r)] for r in range(5)] == eager
    assert len({tuple(x) for x in eager}) == 5
    # the last layer of the last step
    cache, used = dec.caches[-1], [n + 7 for n in lengths]
    q = dec.q.view(5, _SHAPE.heads, _SHAPE.head_dim)
    _check_attention(cache, q, dec.attn.view_as(q), used, dec.window, dec.first_tokens)
    for b in range(5):
        for n, x in ((0, dec.k), (1, dec.v)):
            codes, st, mn = step_ref.quantize(x[b].view(_SHAPE.kv_heads, -1).double().cpu().numpy(), cache.group_size)
            held = _held(cache, b)[n]
            assert np.array_equal(held[0][:, used[b] - 1], codes) and np.array_equal(held[1][:, used[b] - 1], st)
        token, share = step_ref.sample(dec.logits[b].double().cpu().numpy(), uniforms[-1, b].item(), dec.temperature[b].item(),
                                       int(dec.top_k[b]), dec.top_p[b].item(), dec.min_p[b].item())
        assert token == eager[b][-1] == dec.tokens[b].item()
        assert abs(dec.probs[b].item() - share) <= share * 2.0 ** -22
    assert dec.greedy[0].item() == eager[0][-1]               # temperature 0 is the argmax


def test_batch_decoder_refusals(device, model):
    dec = _decoder(device, model, 2, 32)
    u = torch.zeros((3, 2), device=device)
    for bad in (([1], [0, 0], u), ([1, 2], [0, 32], u), ([1, 2], [0, 30], u), ([1, 2], [0, 0], u[:, :1]), ([1, 2], [0, 0], u.double())):
        with pytest.raises(ValueError):
            dec.generate(*bad)
    for batch in (0, 65):
        with pytest.raises(ValueError):
            _decoder(device, model, batch)
    # a request at the capacity's end: further tokens are not stored, nothing else is touched
    dec.prime([3, 4], [31, 5])
    for _ in range(3):
        dec.step()
    assert dec.positions.tolist() == [34, 8]


def test_decoders_that_share_a_backend(device, model):
    """A graph keeps the scratch that it was captured with when a larger batch makes the backend replace
    it: memory that is handed out afterwards is left alone, and the graph's results stay."""
    lengths, u = [40, 1, 33], torch.full((4, 3), 0.4, device=device)
    small = _decoder(device, model, 3)
    _prior(small, [0, 1, 2], lengths)
    want = small.generate([5, 17, 900], lengths, u)
    large = DenseBatchDecoder(small.be, model, 64, 64)
    large.capture()
    assert small._graph_scratch.data_ptr() != large._graph_scratch.data_ptr()
    later = [torch.full((small._graph_scratch.numel(),), 7, device=device, dtype=torch.int64) for _ in range(8)]
    for _ in range(2):
        assert small.generate([5, 17, 900], lengths, u) == want
    assert all(bool((x == 7).all()) for x in later)


def test_token_minus_one(device, model):
    """A request whose logits leave nothing gets token -1; the others get what they would without it."""
    lengths, u = [40, 1, 33], torch.full((3,), 0.4, device=device)
    runs = []
    for spoil in (False, True):
        dec = _decoder(device, model, 3)
        _prior(dec, [0, 1, 2], lengths)
        dec.prime([5, 17, 900], lengths)
        dec.uniforms.copy_(u)
        dec.set_sampling(0.9)
        tokens = []
        for step in range(3):
            if spoil and step == 1:
                dec.tokens[1] = -1
            dec.step()
            tokens.append(dec.tokens.tolist())
        runs.append(tokens)
    assert [t[::2] for t in runs[0]] == [t[::2] for t in runs[1]]


def _chain(be, cache, s):
    be.rotary_rows(s["q"], s["k"], s["pos"], s["freq"], s["qr"], s["kr"])
    be.kv_append_int4(cache, s["kr"], s["v"], s["pos"])
    be.gqa_attention_int4(s["qr"], cache, s["o"], s["len"], window=s["window"], first_tokens=2)
    be.sample_rows(s["logits"], s["u"], s["t"], top_p=s["p"], probs=s["w"])


def _chain_state(device, batch, capacity, seed, window=0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=g, device=device)  # noqa: E731
    freq, _ = rotary_frequencies(64, device=device)
    s = {"q": r(batch, 8, 64).half(), "k": r(batch, 2, 64).half(), "v": r(batch, 2, 64).half(), "freq": freq, "window": window,
         "logits": r(batch, 32000).half() * 3, "u": torch.rand(batch, generator=g, device=device),
         "p": torch.full((batch,), 0.9, device=device), "t": torch.zeros(batch, device=device, dtype=torch.int64),
         "w": torch.zeros(batch, device=device), "pos": torch.randint(40, capacity - 1, (batch,), generator=g, device=device, dtype=torch.int32)}
    s["len"] = s["pos"] + 1
    s["qr"], s["kr"], s["o"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["q"])
    cache = Int4KvCache.allocate(batch, 2, capacity, 64, 32, device)
    return s, cache, (r(batch, capacity, 2, 64).half(), r(batch, capacity, 2, 64).half())


def _fill(be, cache, prior):
    be.kv_append_int4(cache, *prior, torch.zeros(cache.batch, device=cache.device, dtype=torch.int32))


@pytest.mark.parametrize("window", [0, 200])
def test_captured_chains_side_by_side(backend, device, window):
    """Two graphs of the chain over different requests, captured in turn and replayed on two streams at
    once, several times, with eager calls of the same operators in between: each gives its eager result
    every time.  The lengths need the split form with its scratch."""
    want, graphs, states = [], [], []
    for seed in (1, 2):
        s, cache, prior = _chain_state(device, 3, 4096, seed, window)
        _fill(backend, cache, prior)
        _chain(backend, cache, s)
        torch.cuda.synchronize()
        want.append({n: s[n].clone() for n in ("qr", "kr", "o", "t", "w")})
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
            _chain(backend, cache, s)
        graphs.append(graph)
        states.append((s, cache))
    streams = [torch.cuda.Stream(device) for _ in graphs]
    other, other_cache, other_prior = _chain_state(device, 3, 4096, 3, window)
    _fill(backend, other_cache, other_prior)
    _chain(backend, other_cache, other)
    torch.cuda.synchronize()
    eager = {n: other[n].clone() for n in want[0]}
    for round_ in range(4):
        for s, _ in states:
            for n in want[0]:
                s[n].zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            _chain(backend, other_cache, other)           # on the current stream, beside them
        torch.cuda.synchronize()
        for (s, _), w in zip(states, want):
            for n in w:
                assert torch.equal(s[n], w[n]), (round_, n)
        for n in eager:
            assert torch.equal(other[n], eager[n]), (round_, n)


def test_side_stream(backend, device):
    """Calls on another stream than the tensors' own, ordered by events."""
    s, cache, prior = _chain_state(device, 4, 2048, 9)
    _fill(backend, cache, prior)
    _chain(backend, cache, s)
    torch.cuda.synchronize()
    want = {n: s[n].clone() for n in ("qr", "kr", "o", "t", "w")}
    side = torch.cuda.Stream(device)
    for n in want:
        s[n].zero_()
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        _chain(backend, cache, s)
    torch.cuda.current_stream(device).wait_stream(side)
    for n in want:
        assert torch.equal(s[n], want[n]), n


def test_graph_follows_lengths_and_settings(backend, device):
    """One captured attention and one captured sampling follow what their length, position and
    settings tensors hold at each replay, from nothing to the capacity."""
    s, cache, prior = _chain_state(device, 3, 4096, 5)
    _fill(backend, cache, prior)
    logits = s["logits"]
    temperature, top_k = torch.ones(3, device=device), torch.zeros(3, device=device, dtype=torch.int32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
        backend.gqa_attention_int4(s["q"], cache, s["o"], s["len"])
        backend.sample_rows(logits, s["u"], s["t"], temperature=temperature, top_k=top_k, probs=s["w"])
    for lengths, t, k in (([0, 1, 32], 1.0, 0), ([4096, 4095, 33], 0.0, 0), ([800, 0, 2000], 0.5, 3), ([5, 4096, 768], 2.0, 900)):
        s["len"].copy_(torch.tensor(lengths))
        temperature.fill_(t)
        top_k.fill_(k)
        s["o"].fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(cache, s["q"], s["o"], lengths)
        for b in range(3):
            token, _ = step_ref.sample(logits[b].double().cpu().numpy(), s["u"][b].item(), t, k)
            assert s["t"][b].item() == token
