"""What the operators on a paged KV cache refuse, and their restatements on known rows.  Nothing is
launched: every refusal comes before a kernel."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from tests import paged_ref
from thintensor_amd import _lib
from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.paged_cache import PagedKvCache


@pytest.fixture(scope="module")
def be():
    if not _lib.library_path().exists():
        pytest.skip("kernel library not built (run __graft_entry__.build())")
    return HipDecodeBackend(torch.device("cpu"), torch.float16, 64, 64, 64, 64)


def _cache(pages=6, kv_heads=2, page=16, dim=64, dtype=torch.float16, bounds=True):
    return PagedKvCache.allocate(pages, kv_heads, page, dim, dtype, bounds=bounds, device="cpu")


def _f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


# ------------------------------------------------------------------ the cache's bookkeeping
@pytest.mark.parametrize("make", [
    lambda: PagedKvCache(_f16(4, 2, 16), _f16(4, 2, 16)),
    lambda: PagedKvCache(_f16(4, 2, 16, 64), _f16(4, 2, 16, 128)),
    lambda: PagedKvCache(_f16(4, 2, 16, 64).float(), _f16(4, 2, 16, 64).float()),
    lambda: PagedKvCache(_f16(4, 2, 16, 64), _f16(4, 2, 16, 64).bfloat16()),
    lambda: PagedKvCache(_f16(4, 2, 24, 64), _f16(4, 2, 24, 64)),
    lambda: PagedKvCache(_f16(4, 2, 512, 64), _f16(4, 2, 512, 64)),
    lambda: PagedKvCache(_f16(4, 2, 16, 96), _f16(4, 2, 16, 96)),
    lambda: PagedKvCache(_f16(0, 2, 16, 64), _f16(0, 2, 16, 64)),
    lambda: PagedKvCache(_f16(4, 2, 64, 16).transpose(2, 3), _f16(4, 2, 16, 64)),
    lambda: PagedKvCache(_f16(4, 2, 16, 64), _f16(4, 2, 16, 64), _f16(4, 2, 64)),
    lambda: PagedKvCache(_f16(4, 2, 16, 64), _f16(4, 2, 16, 64), _f16(4, 2, 2, 64).bfloat16()),
    lambda: PagedKvCache(_f16(4, 2, 16, 64), _f16(4, 2, 16, 64), _f16(4, 2, 2, 128)[..., :64]),
    lambda: PagedKvCache.allocate(4, 2, 48, 64, device="cpu"), lambda: PagedKvCache.allocate(4, 2, 16, 80, device="cpu"),
    lambda: PagedKvCache.allocate(0, 2, 16, 64, device="cpu")])
def test_cache_refusals(make):
    with pytest.raises(ValueError):
        make()


def test_cache_descriptor():
    both = _f16(5, 16, 2, 3, 64)                              # tokens before K / V before heads
    c = PagedKvCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2))
    assert (c.pages, c.kv_heads, c.page_size, c.head_dim) == (5, 3, 16, 64)
    assert (c.desc.k_page, c.desc.k_head, c.desc.k_token) == (16 * 384, 64, 384)
    assert c.desc.v_pages - c.desc.k_pages == 2 * 192 and c.desc.k_bounds is None
    assert c.nbytes() == both.numel() * 2
    assert _cache().nbytes() == 2 * (2 * 6 * 2 * 16 * 64 + 6 * 2 * 2 * 64)
    with pytest.raises(AttributeError):                       # the descriptor holds the addresses
        c.k_pages = both[:, :, 0].transpose(1, 2).clone()


# ------------------------------------------------------------------ refusals of the backend
def _append_args():
    return {"cache": _cache(), "q": _f16(4, 4, 64), "k": _f16(4, 2, 64), "v": _f16(4, 2, 64), "page_table": _i32(2, 3),
            "starts": _i32(2), "inv_freq": torch.ones(32, dtype=torch.float64)}


@pytest.mark.parametrize("change", [
    {"k": _f16(4, 3, 64)}, {"k": _f16(4, 2, 32)}, {"v": _f16(3, 2, 64)}, {"k": _f16(4, 2, 64).float()}, {"v": _f16(4, 2, 64).bfloat16()},
    {"k": _f16(4, 64, 2).transpose(1, 2)}, {"q": _f16(3, 4, 64)}, {"q": _f16(4, 256)}, {"q": _f16(4, 4, 64).float()},
    {"q": None, "q_out": _f16(4, 4, 64)}, {"q_out": _f16(4, 4, 32)}, {"q_out": _f16(4, 4, 64).bfloat16()},
    {"q_out": _f16(4, 64, 4).transpose(1, 2)}, {"page_table": _i32(3)}, {"page_table": _i32(2, 3).long()},
    {"page_table": _i32(3, 2).t()}, {"page_table": _i32(2, 0)}, {"page_table": _i32(3, 3)}, {"starts": _i32(3)},
    {"starts": _i32(2).long()}, {"cu_tokens": _i32(2)}, {"cu_tokens": _i32(3).long()}, {"page_table": _i32(3, 3), "starts": _i32(3)},
    {"inv_freq": torch.ones(32)}, {"inv_freq": torch.ones(2, 16, dtype=torch.float64)}, {}])
def test_append_refusals(be, change):
    with pytest.raises(ValueError):                           # {}: right, but not on a GPU
        be.rotary_append_paged(**{**_append_args(), **change})


@pytest.mark.parametrize("width,right", [(1, True), (2, False)])
def test_tables_of_one_page_have_any_stride_there(be, width, right):
    table = _i32(3, 2).t()[:, :width]
    assert table.stride() == (1, 2)
    with pytest.raises(ValueError, match="device tensors" if right else "page_table"):
        be.rotary_append_paged(**{**_append_args(), "page_table": table})
    with pytest.raises(ValueError, match="device tensors" if right else "page_table"):
        be.gqa_attention_paged(**{**_attention_args(), "page_table": table})


def _attention_args():
    return {"q": _f16(4, 4, 64), "cache": _cache(), "page_table": _i32(2, 3), "lengths": _i32(2), "out": _f16(4, 4, 64)}


@pytest.mark.parametrize("change", [
    {"q": _f16(4, 256)}, {"q": _f16(4, 4, 64).bfloat16()}, {"out": _f16(4, 4, 64).float()}, {"out": _f16(3, 4, 64)},
    {"q": _f16(4, 3, 64), "out": _f16(4, 3, 64)}, {"q": _f16(4, 4, 128), "out": _f16(4, 4, 128)},
    {"q": _f16(4, 0, 64), "out": _f16(4, 0, 64)}, {"q": _f16(4, 64, 4).transpose(1, 2)}, {"out": _f16(4, 64, 4).transpose(1, 2)},
    {"page_table": _i32(3, 3)}, {"page_table": _i32(2, 3).long()}, {"lengths": _i32(4)}, {"lengths": _i32(2).long()},
    {"cu_tokens": _i32(4)}, {"page_table": _i32(3, 3), "lengths": _i32(3)}, {"sinks": _f16(2)}, {"sinks": _i32(4)},
    {"selected": _i32(2, 2, 2)}, {"selected": _i32(4, 2, 2), "page_table": _i32(4, 3), "lengths": _i32(4), "shared_pages": 1},
    {"selected": _i32(4, 2, 0), "page_table": _i32(4, 3), "lengths": _i32(4)},
    {"selected": _i32(4, 2, 2).long(), "page_table": _i32(4, 3), "lengths": _i32(4)},
    {"selected": _i32(4, 1, 2), "page_table": _i32(4, 3), "lengths": _i32(4)}, {}])
def test_attention_refusals(be, change):
    with pytest.raises(ValueError):
        be.gqa_attention_paged(**{**_attention_args(), **change})


@pytest.mark.parametrize("change", [
    {"q": _f16(2, 256)}, {"q": _f16(2, 3, 64)}, {"q": _f16(2, 4, 64).bfloat16()}, {"q": _f16(3, 4, 64)}, {"q": _f16(2, 64, 4).transpose(1, 2)},
    {"cache": _cache(bounds=False)}, {"page_table": _i32(2, 3).long()}, {"lengths": _i32(3)}, {"selected": _i32(2, 2, 4).long()},
    {"selected": _i32(2, 4)}, {"selected": _i32(2, 1, 4)}, {"selected": _i32(2, 2, 8)[..., ::2]}, {}])
def test_select_refusals(be, change):
    args = {"q": _f16(2, 4, 64), "cache": _cache(), "page_table": _i32(2, 3), "lengths": _i32(2), "selected": _i32(2, 2, 4)}
    with pytest.raises(ValueError):
        be.select_pages(**{**args, **change})


# ------------------------------------------------------------------ refusals of the entry points
_BASE = 1 << 20


def _desc(**change):
    """A cache of addresses that nothing reads."""
    d = dict(k_pages=_BASE, v_pages=_BASE << 4, k_bounds=_BASE << 8, k_page=2048, k_head=1024, k_token=64, v_page=2048,
             v_head=1024, v_token=64, b_page=256, b_head=128, pages=6, kv_heads=2, page_size=16, head_dim=64, dtype=_lib.F16)
    d.update(change)
    return _lib.PagedCache(*[d[n] for n, _ in _lib.PagedCache._fields_])


_BAD_CACHES = [dict(k_pages=None), dict(v_pages=_BASE * 16 + 8), dict(k_bounds=(_BASE << 8) + 2), dict(dtype=_lib.F32), dict(head_dim=96),
               dict(page_size=24), dict(page_size=8), dict(page_size=512), dict(pages=0), dict(pages=1 << 31), dict(kv_heads=0),
               dict(k_token=68), dict(v_head=1028), dict(k_page=2052), dict(b_head=132), dict(k_token=1 << 40)]

_P = 1 << 30


def _call_append(lib, cache=None, **change):
    a = dict(q=_P, qt=256, qh=64, k=_P << 1, kt=128, kh=64, v=_P << 2, vt=128, vh=64, table=_P << 3, tr=3, tp=3, starts=_P << 4,
             cu=None, rows=2, tokens=4, heads=4, f=_P << 5, rotary=64, inter=0, amp=1.0, out=_P, ot=256, oh=64, stream=None)
    a.update(change)
    return lib.tt_rotary_append_paged(cache or _desc(), *a.values())


def _call_attention(lib, cache=None, **change):
    a = dict(q=_P, qt=256, qh=64, table=_P << 3, tr=3, tp=3, lengths=_P << 4, cu=None, rows=2, tokens=4, heads=4, window=0, shared=0,
             sel=None, count=0, limit=48, sinks=None, sd=2, scale=0.125, scratch=None, floats=0, out=_P, ot=256, oh=64, stream=None)
    a.update(change)
    return lib.tt_gqa_attention_paged(cache or _desc(), *a.values())


def _call_select(lib, cache=None, **change):
    a = dict(q=_P, qt=256, qh=64, table=_P << 3, tr=3, tp=3, lengths=_P << 4, rows=2, heads=4, first=1, last=1, limit=48,
             scratch=_P << 5, floats=1 << 20, sel=_P << 6, count=4, stream=None)
    a.update(change)
    return lib.tt_select_pages(cache or _desc(), *a.values())


def test_entry_points_refuse_caches(be):
    for bad in _BAD_CACHES:
        c = _desc(**bad)
        assert _call_append(be.lib, c) == -1, bad
        assert _call_attention(be.lib, c) == -1, bad
        assert _call_select(be.lib, c) == -1, bad
        assert be.lib.tt_select_pages_scratch_floats(c, 3, 2, 48) < 0
        assert be.lib.tt_gqa_attention_paged_scratch_floats(c, 3, 0, 2, 4, 4, 0, 0, 0, 48) < 0
    assert _call_select(be.lib, _desc(k_bounds=None)) == -1


@pytest.mark.parametrize("change", [
    dict(rows=65536), dict(rows=-1), dict(tokens=3), dict(tokens=-2), dict(tokens=(1 << 22) + 2), dict(heads=-2), dict(heads=65536),
    dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(f=None), dict(k=None), dict(v=None), dict(table=None), dict(starts=None),
    dict(q=None), dict(out=None), dict(tp=0), dict(tp=1 << 27),
    dict(out=_P + 2), dict(out=_P << 1), dict(out=(_P << 2) + 128), dict(ot=0), dict(oh=0), dict(out=_BASE), dict(k=_BASE), dict(v=_BASE << 4)])
def test_append_entry_refuses(be, change):
    assert _call_append(be.lib, **change) == -1
    assert be.lib.tt_last_error()


@pytest.mark.parametrize("bad", [dict(k_page=1024), dict(k_head=0), dict(k_token=0), dict(v_pages=_BASE), dict(v_pages=_BASE + 128),
                                 dict(k_bounds=_BASE + 2048), dict(b_page=0), dict(b_head=64), dict(v_token=32)])
def test_append_refuses_caches_that_overlap(be, bad):
    assert _call_append(be.lib, _desc(**bad)) == -1
    assert b"share memory" in be.lib.tt_last_error()


@pytest.mark.parametrize("change", [
    dict(rows=65536), dict(tokens=3), dict(tokens=(1 << 22) + 2), dict(heads=0), dict(heads=3), dict(heads=65536), dict(window=-1),
    dict(limit=0), dict(shared=-1), dict(shared=4), dict(sel=_P << 7), dict(sel=_P << 7, count=2), dict(sel=_P << 7, count=1 << 20, tokens=2),
    dict(sel=_P << 7, count=2, tokens=2, shared=1), dict(sinks=_P << 7, sd=3), dict(scale=math.nan), dict(scale=math.inf),
    dict(q=None), dict(out=None), dict(lengths=None), dict(table=None), dict(tp=0), dict(tp=1 << 27),
    dict(out=_P + 2), dict(ot=0), dict(oh=32), dict(out=_BASE), dict(out=(_BASE << 4) + 512), dict(out=_BASE << 8)])
def test_attention_entry_refuses(be, change):
    assert _call_attention(be.lib, **change) == -1
    assert be.lib.tt_last_error()


@pytest.mark.parametrize("change", [
    dict(rows=65536), dict(heads=0), dict(heads=3), dict(first=-1), dict(last=-1), dict(first=3, last=2), dict(count=0), dict(count=4097),
    dict(limit=0), dict(scratch=None), dict(floats=11), dict(q=None), dict(table=None), dict(lengths=None), dict(sel=None), dict(tp=1 << 27)])
def test_select_entry_refuses(be, change):
    assert _call_select(be.lib, **change) == -1
    assert be.lib.tt_last_error()


@pytest.mark.parametrize("sel", [_P, _P + 2 * 192, (_P << 3) + 20, _P << 4, (_P << 4) + 4, _BASE << 8, _BASE + 4096, (_BASE << 4) + 24000])
def test_selection_shares_no_memory(be, sel):
    assert _call_select(be.lib, sel=sel) == -1
    assert b"share memory" in be.lib.tt_last_error()


def test_nothing_to_do(be):
    for f in (_call_append, _call_attention):
        assert f(be.lib, rows=0, tokens=0) == 0 and f(be.lib, tokens=0) == 0
    assert _call_select(be.lib, rows=0) == 0


def test_an_empty_batch_may_have_a_table_of_no_pages(be):
    c = _desc()
    assert _call_append(be.lib, rows=0, tokens=0, tr=0, tp=0) == 0
    assert be.lib.tt_gqa_attention_paged_scratch_floats(c, 0, 0, 0, 0, 4, 0, 0, 0, 0) == 0
    assert _call_attention(be.lib, rows=0, tokens=0, tr=0, tp=0, limit=0) == 0
    assert be.lib.tt_select_pages_scratch_floats(c, 0, 0, 0) == 0
    assert _call_select(be.lib, rows=0, tr=0, tp=0, limit=0) == 0
    for f in (_call_append, _call_attention, _call_select):
        assert f(be.lib, rows=0, tp=-1, **({} if f is _call_select else dict(tokens=0))) == -1


# ------------------------------------------------------------------ the restatements on known rows
def test_restated_attention_on_known_rows():
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((4, 1, 16, 64)), rng.standard_normal((4, 1, 16, 64))
    q = rng.standard_normal((3, 2, 64))
    table = [[2, 0], [1, 3]]
    out, mag, _, seen, _ = paged_ref.attention(q, k, v, table, [1, 18], [1, 2], 16)
    assert np.allclose(out[0], v[2, 0, 0]) and np.allclose(mag[0], np.abs(v[2, 0, 0])) and list(seen) == [1, 17, 18]
    flat_k, flat_v = np.concatenate((k[1, 0], k[3, 0]))[:18], np.concatenate((v[1, 0], v[3, 0]))[:18]
    p = np.exp(flat_k @ q[2, 1] / 8)
    assert np.allclose(out[2, 1], p @ flat_v / p.sum())
    assert np.allclose(paged_ref.attention(q, k, v, table, [1, 18], [1, 2], 16, window=1)[0][2], flat_v[17])
    sunk = paged_ref.attention(q, k, v, table, [1, 18], [1, 2], 16, sinks=np.zeros(2))[0]
    assert np.allclose(sunk[2, 1], p @ flat_v / (p.sum() + 1))
    one = paged_ref.attention(q[:2], k, v, table, [1, 18], [1, 1], 16, selected=[[[1]], [[1, -1]]])
    assert np.all(one[0][0] == 0) and list(one[3]) == [0, 2]                     # row 0's page 1 holds nothing
    assert np.isnan(paged_ref.attention(q[:1], k, v, [[9]], [3], [1], 16)[0]).all()


def test_restated_selection():
    s = np.array([1, 5, 5, 2, 9, 0], dtype=np.float32)
    assert paged_ref.select(s, 3, 1, 1) == [0, 4, 5]
    assert paged_ref.select(s, 4, 1, 1) == [0, 1, 4, 5]                          # of equal ones the lower
    assert paged_ref.select(s, 8, 2, 3) == [0, 1, 2, 3, 4, 5, -1, -1]
    s[3] = np.nan
    assert paged_ref.select(s, 2, 0, 0) == [3, 4]
    q, b = np.array([[1.0, -2.0]]), np.array([[[[-1.0, 3.0], [2.0, 4.0]]]])
    assert paged_ref.scores(q, b, [0], 1)[0, 0] == 2.0 - 6.0
