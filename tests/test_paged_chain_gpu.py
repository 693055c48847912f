"""The operators on a paged cache as a serving program uses them: a prompt in chunks, steps of a batch in a
captured graph, requests that branch off one prompt, steps over selected pages, graphs side by side and side
streams.  Attention is checked against float64 from what the cache holds, the cache against ``rotary_rows``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.paged_ref import attention, attention_bound, np64, same_bits, scores, select
from thintensor_amd.paged_cache import PagedKvCache

pytestmark = pytest.mark.gpu

_H, _KVH, _D, _PAGE = 8, 2, 64, 16


class Layer:
    """One layer's cache with rows of requests, their lengths on the device."""

    def __init__(self, backend, device, tables, dtype=torch.float16, page=_PAGE, pages=40):
        self.be, self.device, self.dtype = backend, device, dtype
        self.cache = PagedKvCache.allocate(pages, _KVH, page, _D, dtype, bounds=True, device=device)
        self.cache.v_pages.fill_(float("nan"))                  # whatever is read has been written
        self.table = torch.tensor(tables, device=device, dtype=torch.int32)
        self.rows = len(tables)
        self.held = torch.zeros(self.rows, device=device, dtype=torch.int32)
        self.inv_freq = 10000.0 ** (-torch.arange(0, _D, 2, device=device, dtype=torch.float64) / _D)

    def feed(self, q, k, v, out, counts=None, **kw):
        """New tokens: as many for every row, or `counts` of them."""
        each = q.shape[0] // self.rows
        cu = None
        new = torch.full_like(self.held, each)
        if counts is not None:
            new = torch.tensor(counts, device=self.device, dtype=torch.int32)
            cu = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0).to(torch.int32)))
        self.be.rotary_append_paged(self.cache, q, k, v, self.table, self.held, self.inv_freq, cu_tokens=cu)
        self.held.add_(new)
        self.be.gqa_attention_paged(q, self.cache, self.table, self.held, out, cu_tokens=cu, **kw)
        return out

    def step(self, q, k, v, out, selected=None, **kw):
        self.be.rotary_append_paged(self.cache, q, k, v, self.table, self.held, self.inv_freq)
        self.held.add_(1)
        if selected is not None:
            self.be.select_pages(q, self.cache, self.table, self.held, selected, first_pages=1, last_pages=1)
        self.be.gqa_attention_paged(q, self.cache, self.table, self.held, out, selected=selected, **kw)

    def check(self, q, out, counts=None, selected=None):
        """`out` is what queries q (rotated) see of the cache."""
        lengths = self.held.tolist()
        counts = counts or [q.shape[0] // self.rows] * self.rows
        want, mag, reach, seen, peak = attention(np64(q), np64(self.cache.k_pages), np64(self.cache.v_pages), self.table.tolist(), lengths, counts,
                                                 self.cache.page_size, selected=None if selected is None else selected.tolist())
        off = np.abs(np64(out) - want) - attention_bound(want, mag, reach, seen, peak, q.dtype)
        assert np.isfinite(want).all() and off.max() <= 0, float(off.max())


def _tokens(g, n, dtype=torch.float16):
    return [torch.randn((n, h, _D), generator=g, device=g.device).to(dtype) for h in (_H, _KVH, _KVH)]


def test_prompts_in_chunks_then_steps(backend, device):
    g = torch.Generator(device=device).manual_seed(1)
    layer = Layer(backend, device, [[0, 5, 9, 12, 30, 31], [7, 3, 2, 20, 21, 22], [1, 4, 6, 8, 10, 11]])
    for counts in ([40, 1, 17], [3, 0, 31], [1, 1, 1], [20, 5, 0]):
        q, k, v = _tokens(g, sum(counts))
        start = layer.held.tolist()
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(start, counts)]).to(device)
        q0, k0 = backend.rotary_rows(q.clone(), k.clone(), pos, layer.inv_freq)
        out = layer.feed(q, k, v, torch.empty_like(q), counts)
        assert same_bits(q, q0)
        at = 0
        for r, (s, n) in enumerate(zip(start, counts)):
            for i in range(n):
                page, slot = int(layer.table[r, (s + i) // _PAGE]), (s + i) % _PAGE
                assert same_bits(layer.cache.k_pages[page, :, slot], k0[at]) and same_bits(layer.cache.v_pages[page, :, slot], v[at])
                at += 1
        layer.check(q, out, counts)
    assert layer.held.tolist() == [64, 7, 49]


@pytest.mark.parametrize("selected", [False, True])
def test_steps_in_a_graph(backend, device, selected):
    """A captured step, replayed with other inputs, equals the same steps taken one by one."""
    g = torch.Generator(device=device).manual_seed(2)
    tables = [[3, 1, 4, 15, 9, 2, 6, 5], [35, 8, 7, 32, 30, 28, 10, 11], [20, 21, 22, 23, 24, 25, 26, 27]]
    a, b = Layer(backend, device, tables), Layer(backend, device, tables)
    prompt = [61, 30, 95]
    q, k, v = _tokens(g, sum(prompt))
    for layer in (a, b):
        layer.feed(q.clone(), k, v, torch.empty_like(q), prompt)
    bufs = [torch.empty((3, h, _D), device=device, dtype=torch.float16) for h in (_H, _KVH, _KVH, _H)]
    sel = torch.empty((3, _KVH, 4), device=device, dtype=torch.int32) if selected else None
    warm = torch.cuda.Stream(device)
    keep = [t.clone() for t in (a.cache.k_pages, a.cache.v_pages, a.cache.k_bounds, a.held)]
    for t in bufs[:3]:
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=warm):
        a.step(*bufs, selected=sel)
    for t, s in zip((a.cache.k_pages, a.cache.v_pages, a.cache.k_bounds, a.held), keep):
        t.copy_(s)
    for step in range(20):
        q, k, v = _tokens(g, 3)
        for t, s in zip(bufs, (q, k, v)):
            t.copy_(s)
        graph.replay()
        out = torch.empty_like(q)
        sel_b = torch.empty_like(sel) if selected else None
        b.step(q, k, v, out, selected=sel_b)
        torch.cuda.synchronize()
        assert same_bits(bufs[3], out) and same_bits(bufs[0], q) and torch.equal(a.held, b.held), step
        assert same_bits(a.cache.k_pages, b.cache.k_pages) and same_bits(a.cache.k_bounds, b.cache.k_bounds)
        if selected:
            assert torch.equal(sel, sel_b)
            bounds = np64(b.cache.k_bounds)
            for r, n in enumerate(b.held.tolist()):
                s = scores(np64(q[r]), bounds, tables[r], -(-n // _PAGE))
                assert [select(x, 4, 1, 1) for x in s] == sel_b[r].tolist()
        b.check(q, out, selected=sel_b)
    for r, n in enumerate(b.held.tolist()):                     # bounds have followed all along
        for p in range(-(-n // _PAGE)):
            page, m = tables[r][p], min(_PAGE, n - p * _PAGE)
            keys = b.cache.k_pages[page, :, :m]
            assert same_bits(b.cache.k_bounds[page], torch.stack((keys.amin(1), keys.amax(1)), 1))


def test_requests_that_branch_off_one_prompt(backend, device):
    """Five requests share a prompt's whole pages; each gets tokens of its own.  Reading the prompt once is reading it
    five times."""
    g = torch.Generator(device=device).manual_seed(3)
    prompt, shared = 83, 83 // _PAGE
    tables = [[10, 4, 7, 1, 0, 20 + 3 * r, 21 + 3 * r, 22 + 3 * r] for r in range(5)]
    layer = Layer(backend, device, tables, torch.bfloat16)
    first = Layer(backend, device, tables[:1], torch.bfloat16)
    first.cache, first.held = layer.cache, torch.zeros_like(first.held)
    q, k, v = _tokens(g, prompt, torch.bfloat16)
    first.feed(q, k, v, torch.empty_like(q), [prompt])
    for r in range(1, 5):                                       # the page that the prompt fills in part is copied
        for t in (layer.cache.k_pages, layer.cache.v_pages, layer.cache.k_bounds):
            t[tables[r][5]] = t[tables[0][5]]
    layer.held.fill_(prompt)
    for step in range(8):
        q, k, v = _tokens(g, 5, torch.bfloat16)
        out = torch.empty_like(q)
        layer.step(q, k, v, out, shared_pages=shared)
        layer.check(q, out)
    q, k, v = _tokens(g, 5 * 6, torch.bfloat16)                  # drafts
    out = layer.feed(q, k, v, torch.empty_like(q), shared_pages=shared)
    layer.check(q, out)


def test_graphs_side_by_side(backend, device):
    """Two captured calls that need scratch, replayed at the same time on two streams, and an eager one between."""
    g = torch.Generator(device=device).manual_seed(4)
    calls = []
    for rows, pages, tokens, shared in ((2, 120, 1, 0), (9, 40, 2, 30)):
        cache = PagedKvCache.allocate(pages * (1 if shared else rows) + rows * 20, _KVH, 64, 128, torch.bfloat16, device=device)
        cache.k_pages.normal_(generator=g)
        cache.v_pages.normal_(generator=g)
        table = torch.randint(0, cache.pages, (rows, pages), generator=g, device=device, dtype=torch.int32)
        table[:, :shared] = table[:1, :shared]
        lengths = torch.tensor([64 * pages - 5 * r for r in range(rows)], device=device, dtype=torch.int32)
        q = torch.randn((rows * tokens, _H, 128), generator=g, device=device).bfloat16()
        out = torch.empty_like(q)
        calls.append((lambda o=out, q=q, c=cache, t=table, n=lengths, s=shared: backend.gqa_attention_paged(q, c, t, n, o, shared_pages=s), out))
    want = []
    for f, out in calls:
        want.append(f().clone())
    graphs, streams = [], [torch.cuda.Stream(device) for _ in calls]
    torch.cuda.synchronize()
    for (f, _), s in zip(calls, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            f()
        graphs.append(graph)
    for turn in range(6):
        for _, out in calls:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        if turn % 2:
            spare = torch.randn(1 << 20, device=device)          # eager work between
            assert torch.isfinite(spare.sum())
        torch.cuda.synchronize()
        for (_, out), w in zip(calls, want):
            assert same_bits(out, w)


def test_side_streams(backend, device):
    """Everything on a stream that is not the default one, behind work that the default one still does."""
    g = torch.Generator(device=device).manual_seed(5)
    tables = [[3, 1, 4, 15], [9, 2, 6, 5]]
    a, b = Layer(backend, device, tables), Layer(backend, device, tables)
    q, k, v = _tokens(g, 2 * 33)
    out_a = a.feed(q.clone(), k, v, torch.empty_like(q))
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    busy = torch.randn((2048, 2048), device=device)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(side):
        q2 = q.clone()
        out_b = b.feed(q2, k, v, torch.empty_like(q))
    side.synchronize()
    torch.cuda.synchronize()
    assert same_bits(out_a, out_b) and same_bits(a.cache.k_pages, b.cache.k_pages)


def test_the_same_bits_every_time(backend, device):
    """No result depends on which workgroup comes first."""
    g = torch.Generator(device=device).manual_seed(6)
    cache = PagedKvCache.allocate(300, 2, 32, 128, torch.bfloat16, bounds=True, device=device)
    for t in (cache.k_pages, cache.v_pages):
        t.normal_(generator=g)
    cache.k_bounds.copy_(torch.stack((cache.k_pages.amin(2), cache.k_pages.amax(2)), 2))
    table = torch.randperm(300, generator=g, device=device).to(torch.int32)[:280].view(4, 70).contiguous()
    lengths = torch.tensor([2240, 1999, 64, 1500], device=device, dtype=torch.int32)
    for tokens in (1, 90):
        q = torch.randn((4 * tokens, 8, 128), generator=g, device=device).bfloat16()
        outs = [backend.gqa_attention_paged(q, cache, table, lengths, torch.empty_like(q), shared_pages=s) for s in (0, 0, 0)]
        assert same_bits(outs[0], outs[1]) and same_bits(outs[0], outs[2])
    q = torch.randn((4, 8, 128), generator=g, device=device).bfloat16()
    picks = [backend.select_pages(q, cache, table, lengths, torch.empty((4, 2, 20), device=device, dtype=torch.int32)) for _ in range(3)]
    assert torch.equal(picks[0], picks[1]) and torch.equal(picks[0], picks[2])
