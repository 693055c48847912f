"""What the operators of a decode step around its weights refuse, their frequencies and the 4-bit
cache's bookkeeping.  Nothing is launched: every refusal comes before a kernel."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from tests import step_ref
from thintensor_amd import _lib
from thintensor_amd.backend import HipDecodeBackend
from thintensor_amd.kv_cache import Int4KvCache
from thintensor_amd.rotary import rotary_frequencies


@pytest.fixture(scope="module")
def be():
    if not _lib.library_path().exists():
        pytest.skip("kernel library not built (run __graft_entry__.build())")
    return HipDecodeBackend(torch.device("cpu"), torch.float16, 64, 64, 64, 64)


def _cache(batch=2, kv_heads=2, capacity=64, head_dim=64, group=32):
    return Int4KvCache.allocate(batch, kv_heads, capacity, head_dim, group, device="cpu")


# ------------------------------------------------------------------ rotary
def test_frequencies():
    f, a = rotary_frequencies(64, 10000.0, device="cpu")
    assert a == 1.0 and f.dtype == torch.float64
    np.testing.assert_allclose(f.numpy(), [10000.0 ** (-2 * i / 64) for i in range(32)], rtol=1e-14)
    lin, _ = rotary_frequencies(64, 10000.0, scaling="linear", factor=4.0, device="cpu")
    np.testing.assert_allclose(lin.numpy(), f.numpy() / 4, rtol=1e-14)
    ntk, _ = rotary_frequencies(64, 10000.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and math.isclose(ntk[-1].item(), f[-1].item() / 4, rel_tol=1e-12)
    yarn, a = rotary_frequencies(64, 150000.0, scaling="yarn", factor=32.0, original_positions=4096, device="cpu")
    base, _ = rotary_frequencies(64, 150000.0, device="cpu")
    assert math.isclose(a, 0.1 * math.log(32.0) + 1.0)
    ratio = (yarn / base).numpy()
    assert ratio[0] == 1.0 and math.isclose(ratio[-1], 1 / 32, rel_tol=1e-12) and np.all(np.diff(ratio) <= 0)
    bands, _ = rotary_frequencies(128, 500000.0, scaling="bands", factor=8.0, original_positions=8192, device="cpu")
    base, _ = rotary_frequencies(128, 500000.0, device="cpu")
    wave = 2 * math.pi / base.numpy()
    ratio = (bands / base).numpy()
    assert np.all(ratio[wave < 8192 / 4] == 1.0) and np.allclose(ratio[wave > 8192], 1 / 8)
    for bad in (dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, scaling="other"), dict(rotary_dim=64, factor=0.5),
                dict(rotary_dim=64, theta=0.0), dict(rotary_dim=64, scaling="bands", low_freq_factor=4.0),
                dict(rotary_dim=64, factor=math.nan), dict(rotary_dim=64, theta=math.inf),
                dict(rotary_dim=64, theta=1.0, scaling="yarn"), dict(rotary_dim=64, scaling="yarn", original_positions=0),
                dict(rotary_dim=64, scaling="yarn", beta_slow=0.0), dict(rotary_dim=64, scaling="yarn", beta_fast=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad, device="cpu")


def _rotary_args():
    return {"q": torch.zeros(3, 4, 64, dtype=torch.float16), "k": torch.zeros(3, 2, 64, dtype=torch.float16),
            "positions": torch.zeros(3, dtype=torch.int32), "inv_freq": torch.ones(32, dtype=torch.float64)}


@pytest.mark.parametrize("change", [
    {"q": torch.zeros(3, 256, dtype=torch.float16)}, {"k": torch.zeros(2, 2, 64, dtype=torch.float16)},
    {"k": torch.zeros(3, 2, 64)}, {"k": torch.zeros(3, 2, 32, dtype=torch.float16)},
    {"positions": torch.zeros(2, dtype=torch.int32)}, {"positions": torch.zeros(3)},
    {"inv_freq": torch.ones(32)}, {"inv_freq": torch.ones(2, 16, dtype=torch.float64)},
    {"q": torch.zeros(3, 64, 4, dtype=torch.float16).transpose(1, 2)},
    {"q_out": torch.zeros(3, 4, 32, dtype=torch.float16)}, {"q_out": torch.zeros(3, 4, 64)},
    {"k": None, "k_out": torch.zeros(3, 2, 64, dtype=torch.float16)}, {}])
def test_rotary_refusals(be, change):
    with pytest.raises(ValueError):                    # {}: right, but not on a GPU
        be.rotary_rows(**{**_rotary_args(), **change})


def test_rotary_entry_refuses_sizes(be):
    one = ctypes.c_void_p(1 << 20)
    f = lambda **c: be.lib.tt_rotary_rows(*[{**dict(  # noqa: E731
        q=one, qt=0, qh=0, k=one, kt=0, kh=0, dt=0, pos=one, pb=4, f=one, a=1.0, i=0, t=1, h=1, kv=1, d=64, r=64,
        qo=one, qot=0, qoh=0, ko=one, kot=0, koh=0, st=None), **c}[n] for n in
        "q qt qh k kt kh dt pos pb f a i t h kv d r qo qot qoh ko kot koh st".split()])
    for c in (dict(t=-1), dict(h=0), dict(kv=-1), dict(r=63), dict(r=0), dict(r=66), dict(d=0), dict(dt=3), dict(pb=2),
              dict(q=None), dict(f=None), dict(ko=None), dict(d=2048)):
        assert f(**c) == -1, c
    assert f(t=0) == 0 and f(t=0, q=None) == 0         # nothing to do


# ------------------------------------------------------------------ the cache
def test_cache_shapes():
    c = _cache(3, 2, 100, 128, 64)
    assert (c.batch, c.kv_heads, c.capacity, c.head_dim, c.group_size) == (3, 2, 128, 128, 64)
    assert c.nbytes() == 3 * 2 * 128 * (128 + 8 * 2)
    part = c.sequences(1, 3)
    assert part.batch == 2 and part.k_codes.data_ptr() == c.k_codes[1].data_ptr()
    for bad in ((0, 2, 64, 64, 32), (1, 0, 64, 64, 32), (1, 1, 0, 64, 32), (1, 1, 64, 96, 32), (1, 1, 64, 64, 128),
                (1, 1, 64, 64, 16)):
        with pytest.raises(ValueError):
            _cache(*bad)
    for a, b in ((2, 2), (-1, 1), (1, 4)):
        with pytest.raises(ValueError):
            c.sequences(a, b)
    t = (c.k_codes, c.k_scales, c.v_codes, c.v_scales)
    for i, bad in ((0, c.k_codes.to(torch.int64)), (1, c.k_scales.float()), (2, c.v_codes[:, :, :-1]), (3, c.v_scales[:, :1]),
                   (0, c.k_codes[:, :, ::2]), (0, c.k_codes[:0]), (1, c.k_scales[:, :, :, :1]), (0, c.k_codes[0]), (3, c.v_scales.transpose(3, 4))):
        with pytest.raises(ValueError):
            Int4KvCache(*[bad if i == j else x for j, x in enumerate(t)])


def test_steps_have_seven_bits():
    s = step_ref.steps()
    m, _ = np.frexp(s)
    assert np.all(m * 128 == np.rint(m * 128)) and np.all(s.astype(np.float16).astype(np.float64) == s)
    codes = np.arange(16)[:, None] * s
    assert np.all(codes.astype(np.float16).astype(np.float64) == codes)      # what the matrix cores take


def _kv(rows=2, tokens=3, kv_heads=2, dim=64, dtype=torch.float16):
    return torch.zeros(rows, tokens, kv_heads, dim, dtype=dtype)


@pytest.mark.parametrize("name", ["kv_append_int4", "kv_read_int4"])
def test_kv_rows_refusals(be, name):
    op, c, starts = getattr(be, name), _cache(), torch.zeros(2, dtype=torch.int32)
    ok = _kv()
    for k, v, s, n in (
            (_kv(3), _kv(3), torch.zeros(3, dtype=torch.int32), None), (_kv(kv_heads=1), _kv(kv_heads=1), starts, None),
            (_kv(dim=128), _kv(dim=128), starts, None), (ok, _kv(tokens=2), starts, None),
            (ok, _kv(dtype=torch.bfloat16), starts, None), (ok, ok, starts.long(), None), (ok, ok, starts[:1], None),
            (ok, ok, starts, torch.zeros(2)), (ok[0, 0], ok[0, 0], starts, None),
            (ok.transpose(2, 3).contiguous().transpose(2, 3), ok, starts, None), (ok, ok, starts, None)):
        with pytest.raises(ValueError):
            op(c, k, v, s, n)


def test_append_refuses_shared_memory(be):
    """Sequences or heads of stride 0 may be read, not written; calls that write nothing pass."""
    c, one = _cache(), ctypes.c_void_p(1 << 20)
    call = lambda d, rows=2, tokens=1: be.lib.tt_kv_append_int4(d, one, 0, 0, 0, one, 0, 0, 0, 0, one, None, rows, tokens, None)  # noqa: E731
    for field in ("kc_seq", "ks_seq", "vc_seq", "vs_seq", "kc_head", "ks_head", "vc_head", "vs_head"):
        d = _lib.Int4Cache.from_buffer_copy(c.desc)
        setattr(d, field, 0)
        assert call(d) == -1 and b"share" in be.lib.tt_last_error(), field
        assert call(d, rows=0) == 0 and call(d, tokens=0) == 0


def test_attention_refusals(be):
    c, q, n = _cache(), torch.zeros(2, 4, 64, dtype=torch.float16), torch.ones(2, dtype=torch.int32)
    good = dict(q=q, cache=c, out=torch.zeros_like(q), lengths=n)
    for change in (dict(q=q[0]), dict(out=q[:1]), dict(out=q.float()), dict(q=q.float(), out=q.float()),
                   dict(q=q[:, :3], out=q[:, :3]), dict(q=q[..., :32], out=q[..., :32]), dict(lengths=n.long()),
                   dict(lengths=n[:1]), dict(sinks=torch.zeros(3)), dict(cache=_cache(1)), {}):
        with pytest.raises(ValueError):
            be.gqa_attention_int4(**{**good, **change})


def test_attention_entry_refuses_sizes(be):
    c = _cache()
    need = lambda *a: be.lib.tt_gqa_attention_int4_scratch_floats(*a)  # noqa: E731
    assert need(c.desc, 2, 4, 0, 0, 64) == 0
    for a in ((3, 4, 0, 0, 64), (2, 3, 0, 0, 64), (2, 4, -1, 0, 64), (2, 4, 0, -1, 64), (2, 4, 0, 0, 0), (2, 0, 0, 0, 64)):
        assert need(c.desc, *a) == -1, a
    long = _cache(1, 1, 1 << 16)
    floats = need(long.desc, 1, 4, 0, 0, 1 << 16)
    assert floats > 0 and need(long.desc, 1, 4, 100, 4, 1 << 16) < floats
    one = ctypes.c_void_p(1 << 20)
    call = lambda dt, scratch, n, length=one: be.lib.tt_gqa_attention_int4(  # noqa: E731
        long.desc, one, 0, 0, dt, length, 1, 4, 0, 0, 1 << 16, None, 0, 1.0, scratch, n, one, 0, 0, None)
    assert call(0, None, 0) == -1 and call(0, one, floats - 1) == -1 and call(2, one, floats) == -1
    assert call(0, one, floats, None) == -1
    for scale in (float("nan"), float("inf")):
        assert be.lib.tt_gqa_attention_int4(long.desc, one, 0, 0, 0, one, 1, 4, 0, 0, 1 << 16, None, 0, scale, one, floats, one,
                                            0, 0, None) == -1
    for field, value in (("capacity", 48), ("head_dim", 96), ("group_size", 16), ("k_codes", None), ("kv_heads", 0),
                         ("kc_head", 2), ("vs_seq", 4), ("v_codes", (1 << 20) + 8)):
        d = _lib.Int4Cache.from_buffer_copy(c.desc)
        setattr(d, field, value)
        assert need(d, 2, 4, 0, 0, 64) == -1, field


# ------------------------------------------------------------------ sampling
def test_sample_refusals(be):
    x, u, t = torch.zeros(2, 50), torch.zeros(2), torch.zeros(2, dtype=torch.int64)
    good = dict(logits=x, uniforms=u, tokens=t)
    for change in (dict(logits=x[0]), dict(logits=x.t()), dict(logits=x[:, :0]), dict(uniforms=u.double()), dict(uniforms=u[:1]),
                   dict(tokens=t.int()), dict(tokens=t[:1]), dict(temperature=u.half()), dict(temperature=u[:1]),
                   dict(top_k=t), dict(top_p=t.int()), dict(min_p=torch.zeros(3)), dict(probs=u.double()), {}):
        with pytest.raises(ValueError):
            be.sample_rows(**{**good, **change})


def test_sample_entry_refuses_sizes(be):
    one = ctypes.c_void_p(1 << 20)
    need = be.lib.tt_sample_rows_scratch_bytes(3, 1000)
    assert need > 0 and be.lib.tt_sample_rows_scratch_bytes(-1, 1000) < 0
    call = lambda **c: be.lib.tt_sample_rows(*[{**dict(x=one, s=1000, dt=2, r=3, v=1000, u=one, a=None, b=None, c=None,  # noqa: E731
                                                       d=None, w=one, n=need, t=one, p=None, st=None), **c}[k]
                                               for k in "x s dt r v u a b c d w n t p st".split()])
    for c in (dict(r=-1), dict(v=0), dict(v=(1 << 20) + 1), dict(dt=4), dict(x=None), dict(u=None), dict(t=None), dict(w=None),
              dict(n=need - 1), dict(w=ctypes.c_void_p(8)), dict(r=65536, n=1 << 40)):
        assert call(**c) == -1, c
    assert call(r=0, x=None) == 0


def test_sample_reference_on_known_rows():
    x = [0.0, math.log(2.0), math.log(5.0), -math.inf]           # weights 1, 2, 5
    assert [step_ref.sample(x, u)[0] for u in (0.0, 0.62, 0.63, 0.87, 0.88)] == [2, 2, 1, 1, 0]
    assert step_ref.sample(x, 0.99, top_k=1) == (2, 1.0) and step_ref.sample(x, 0.99, temperature=0.0) == (2, 1.0)
    assert step_ref.sample(x, 0.99, top_p=0.6)[0] == 2 and step_ref.sample(x, 0.99, top_p=0.7)[0] == 1
    assert step_ref.sample(x, 0.99, min_p=0.3)[0] == 1 and step_ref.sample([-math.inf], 0.5) == (-1, 0.0)
    assert step_ref.sample([1.0, 3.0, 3.0], 0.0)[0] == 1
