"""The host's checks of operands that share memory: the rule against sets of bytes, and what the entry
points refuse by it.  Nothing is launched."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from thintensor_amd import _lib
from thintensor_amd.backend import HipDecodeBackend

_CSRC = Path(__file__).resolve().parents[1] / "thintensor_amd" / "csrc"

_PROGRAM = r"""
#include <cstdio>
#include "tt_regions.h"
// lines of: element, then twice start, length, three times (elements, stride)
int main() {
  long v[17];
  for (;;) {
    for (int i = 0; i < 17; i++)
      if (scanf("%ld", &v[i]) != 1) return 0;
    const auto make = [&](const long* p) {
      return tt::Region(reinterpret_cast<const void*>(p[0]), v[0], p[1], {{p[2], p[3]}, {p[4], p[5]}, {p[6], p[7]}});
    };
    const tt::Region a = make(v + 1), b = make(v + 9);
    printf("%d %d %d\n", a.once(), apart(a, b), a.same(b));
  }
}
"""


def _bytes(element, start, length, axes):
    at = [start]
    for n, stride in axes:
        at = [x + i * stride * element for x in at for i in range(n)]
    return [x + i for x in at for i in range(element * length)]


def _run(tmp_path, cases):
    compiler = shutil.which("g++") or shutil.which("clang++")
    if compiler is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "regions.cpp").write_text(_PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O1", "-I", str(_CSRC), str(tmp_path / "regions.cpp"), "-o", str(tmp_path / "regions")],
                   check=True)
    lines = [" ".join(map(str, [e, *(x for p, n, axes in (a, b) for x in (p, n, *(y for ax in axes for y in ax)))])) for e, a, b in cases]
    out = subprocess.run([str(tmp_path / "regions")], input="\n".join(lines), capture_output=True, text=True, check=True).stdout
    return [tuple(int(x) for x in line.split()) for line in out.splitlines()]


def test_rule_against_sets_of_bytes(tmp_path):
    """What passes has no byte twice and none in common; heads of tokens, side by side in a row as the parts
    of a QKV row are, are told apart exactly."""
    rng = random.Random(5)
    cases = []
    for _ in range(4000):
        def region():
            axes = [(rng.choice([0, 1, 2, 3, 5]) if rng.random() < 0.3 else rng.randint(1, 4), rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, -4, -12, 48]))
                    for _ in range(3)]
            return 4096 + rng.randint(-60, 60), rng.randint(1, 4), axes
        cases.append((rng.choice([2, 4]), region(), region()))
    rows = []
    for _ in range(2000):                      # two parts of rows of `width` elements, contiguous heads of `dim`
        dim, width, tokens = rng.randint(1, 3), rng.randint(8, 14), rng.randint(1, 4)
        a, b = rng.randint(1, 3), rng.randint(1, 3)
        off = [rng.randint(0, max(0, width - n * dim)) for n in (a, b)]
        rows.append((2, (4096 + 2 * off[0], dim, [(1, 0), (tokens, width), (a, dim)]), (4096 + 2 * off[1], dim, [(1, 7), (tokens, width), (b, dim)])))
    got = _run(tmp_path, cases + rows)
    assert len(got) == 6000
    kept = [0, 0]
    for (e, a, b), (once, apart, same) in zip(cases, got):
        sa, sb = _bytes(e, *a), _bytes(e, *b)
        if once:
            assert len(set(sa)) == len(sa), a
        if apart:
            assert not set(sa) & set(sb), (e, a, b)
        if same:
            assert sorted(set(sa)) == sorted(set(sb)), (a, b)
        kept[0] += once
        kept[1] += apart
    assert min(kept) > 400
    for (e, a, b), (once, apart, _) in zip(rows, got[4000:]):
        sa, sb = _bytes(e, *a), _bytes(e, *b)
        assert bool(once) == (len(set(sa)) == len(sa)) and bool(apart) == (not set(sa) & set(sb)), (a, b)


@pytest.fixture(scope="module")
def be():
    if not _lib.library_path().exists():
        pytest.skip("kernel library not built (run __graft_entry__.build())")
    return HipDecodeBackend(torch.device("cpu"), torch.float16, 64, 64, 64, 64)


_AT = 1 << 20                                   # (bytes)


@pytest.mark.parametrize("change", [
    dict(qot=0), dict(qoh=0), dict(qoh=32), dict(qot=64),                      # an output's tokens or heads in one place
    dict(kot=0), dict(koh=0), dict(kot=2 * 64 - 8),
    dict(ko=_AT + (1 << 16)), dict(ko=_AT + (1 << 16) + 2 * 3 * 64), dict(ko=_AT + (1 << 16) + 2 * 2 * 4 * 64 + 2),   # both outputs
    dict(qo=_AT + 2), dict(qo=_AT + 2 * 4 * 64), dict(qo=_AT, qot=8 * 64),        # an output across its input
    dict(qo=_AT + (2 << 16)), dict(ko=_AT), dict(ko=_AT + 2 * 9 * 64),            # ... and the other input
    dict(qt=0, qo=_AT, qot=0)])                                                 # an expanded tensor in place
def test_rotary_refuses_shared_memory(be, change):
    """Three tokens of four query heads and two KV heads of 64 dims, elements of two bytes."""
    args = dict(q=_AT, qt=4 * 64, qh=64, k=_AT + (2 << 16), kt=2 * 64, kh=64, dt=0, pos=64, pb=4, f=64, a=1.0, i=0, t=3, h=4,
                kv=2, d=64, r=64, qo=_AT + (1 << 16), qot=4 * 64, qoh=64, ko=_AT + (3 << 16), kot=2 * 64, koh=64, st=None)
    args.update(change)
    point = lambda n, x: ctypes.c_void_p(x) if n in ("q", "k", "pos", "f", "qo", "ko") else x  # noqa: E731
    rc = be.lib.tt_rotary_rows(*[point(n, args[n]) for n in "q qt qh k kt kh dt pos pb f a i t h kv d r qo qot qoh ko kot koh st".split()])
    assert rc == -1 and b"memory" in be.lib.tt_last_error(), be.lib.tt_last_error()


def _desc(rows=3, kv_heads=2, capacity=64, head_dim=64, group=32, **change):
    """Arrays far from each other, sequences and heads one after the other."""
    words, pairs = capacity * head_dim // 8, capacity * head_dim // group * 2
    d = _lib.Int4Cache(*[_AT + (i << 20) for i in range(4)], kv_heads * words, words, kv_heads * pairs, pairs, kv_heads * words,
                       words, kv_heads * pairs, pairs, rows, kv_heads, capacity, head_dim, group)
    for n, x in change.items():
        setattr(d, n, x)
    return d


_WORDS, _PAIRS = 64 * 8, 64 * 2 * 2            # of a sequence and head of _desc(): int32 and fp16 elements


@pytest.mark.parametrize("change", [
    dict(kc_head=_WORDS - 4), dict(vc_head=_WORDS - 4), dict(ks_head=_PAIRS - 8), dict(vs_head=_PAIRS - 8),
    dict(kc_seq=_WORDS), dict(vs_seq=_PAIRS), dict(kc_seq=0, kv_heads=1), dict(v_codes=_AT),
    dict(v_codes=_AT + 4 * 3 * 2 * _WORDS - 16), dict(k_scales=_AT + (3 << 20) + 2 * _PAIRS)])
def test_append_refuses_memory_that_meets(be, change):
    one = ctypes.c_void_p(1 << 30)
    rc = be.lib.tt_kv_append_int4(_desc(**change), one, 128, 0, 64, one, 128, 0, 64, 0, one, None, 3, 1, None)
    assert rc == -1 and b"share" in be.lib.tt_last_error(), be.lib.tt_last_error()


@pytest.mark.parametrize("change", [
    dict(k_token=0), dict(k_head=0), dict(k_row=0), dict(v_row=4 * 128), dict(v_head=32), dict(v_token=64),
    dict(v=1 << 30), dict(v=(1 << 30) + 2 * 64), dict(k=_AT + (2 << 20)), dict(v=_AT + (1 << 20) + 2 * _PAIRS), dict(k=_AT - 4)])
def test_read_refuses_outputs_that_meet(be, change):
    """Three rows of five tokens, two heads of 64 dims, elements of two bytes."""
    a = dict(k=1 << 30, k_row=640, k_token=128, k_head=64, v=1 << 31, v_row=640, v_token=128, v_head=64)
    a.update(change)
    if "v" in change and change["v"] == (1 << 30) + 128:        # v's heads among k's
        a.update(k_token=256, k_row=5 * 256, v_token=256, v_row=5 * 256, k_head=64)
    rc = be.lib.tt_kv_read_int4(_desc(), ctypes.c_void_p(a["k"]), a["k_row"], a["k_token"], a["k_head"], ctypes.c_void_p(a["v"]),
                                a["v_row"], a["v_token"], a["v_head"], 0, ctypes.c_void_p(64), None, 3, 5, None)
    assert rc == -1 and b"share" in be.lib.tt_last_error(), be.lib.tt_last_error()


@pytest.mark.parametrize("change", [
    dict(out_row=0), dict(out_head=0), dict(out_head=60), dict(out_row=200), dict(out=1 << 30, out_row=512),
    dict(out=(1 << 30) + 2 * 64), dict(out=(1 << 30) - 2), dict(out=_AT + (2 << 20)), dict(q_row=0, out=1 << 30, out_row=0)])
def test_attention_refuses_outputs_that_meet(be, change):
    """Three rows of four heads of 64 dims."""
    a = dict(q=1 << 30, q_row=256, q_head=64, out=1 << 31, out_row=256, out_head=64)
    a.update(change)
    rc = be.lib.tt_gqa_attention_int4(_desc(), ctypes.c_void_p(a["q"]), a["q_row"], a["q_head"], 0, ctypes.c_void_p(64), 3, 4, 0, 0, 64,
                                      None, 0, 1.0, None, 0, ctypes.c_void_p(a["out"]), a["out_row"], a["out_head"], None)
    assert rc == -1 and b"share" in be.lib.tt_last_error(), be.lib.tt_last_error()
