"""The alignment that a 4-bit cache's arrays need, array by array: what the header says is taken, less is
refused by a message that names the array.  Nothing is launched."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

from thintensor_amd import _lib

_AT = 1 << 20


@pytest.fixture(scope="module")
def need():
    if not _lib.library_path().exists():
        pytest.skip("kernel library not built (run __graft_entry__.build())")
    lib = _lib.load(build_if_missing=False)
    return lambda d: (lib.tt_gqa_attention_int4_scratch_floats(d, 2, 4, 0, 0, 64), lib.tt_last_error())


def _desc(head_dim, group, **change):
    words, pairs = 64 * head_dim // 8, 64 * head_dim // group * 2
    d = _lib.Int4Cache(*[_AT + (i << 20) for i in range(4)], 2 * words, words, 2 * pairs, pairs, 2 * words, words, 2 * pairs, pairs,
                       2, 2, 64, head_dim, group)
    for n, x in change.items():
        setattr(d, n, x)
    return d


_SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dim,group", _SHAPES)
def test_k_scales(need, dim, group):
    """Two scale pairs are read as one of eight bytes where a quarter of the dims has two groups."""
    size = 8 if (dim, group) == (256, 32) else 4
    at = _AT + (1 << 20)
    for off in (0, 2, 4, 8, 12):
        rc, said = need(_desc(dim, group, k_scales=at + off))
        assert rc == (0 if off % size == 0 else -1), off
        assert rc == 0 or b"k_scales must be %d-byte" % size in said, said
    pairs = 64 * dim // group * 2
    for field in ("ks_seq", "ks_head"):
        for more in (1, 2, 4):
            rc, said = need(_desc(dim, group, **{field: 2 * pairs + more}))
            assert rc == (0 if 2 * more % size == 0 else -1), (field, more)
            assert rc == 0 or b"k_scales" in said and b"%d-byte" % size in said, said


@pytest.mark.parametrize("field,off", [("k_codes", 8), ("v_codes", 4), ("v_scales", 8), ("kc_seq", 2), ("kc_head", 1), ("vc_seq", 2),
                                       ("vc_head", 2), ("vs_seq", 4), ("vs_head", 4)])
def test_other_arrays(need, field, off):
    good = _desc(128, 32)
    rc, said = need(_desc(128, 32, **{field: getattr(good, field) + off}))
    assert rc == -1 and b"16-byte" in said and b"k_scales" not in said, said


def test_header_states_the_rule():
    text = (Path(__file__).resolve().parents[1] / "include" / "thintensor_hip.h").read_text()
    text = re.sub(r"\s+\*?\s*", " ", text)
    assert "k_scales on 8 bytes with head_dim 256 and group_size 32, on 4 otherwise" in text
