"""How a row of the 4-bit cache is shared by workgroups: by the compute units that the GPU says it has."""

from __future__ import annotations

import pytest
import torch

from thintensor_amd.kv_cache import Int4KvCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,kv_heads,heads,tokens", [(1, 1, 4, 65536), (1, 8, 32, 16384), (4, 10, 40, 4064), (2, 8, 64, 131072),
                                                        (64, 8, 8, 65536), (16, 16, 16, 2048), (16, 16, 16, 2080), (1, 1, 48, 768)])
def test_scratch_follows_the_compute_units(backend, device, rows, kv_heads, heads, tokens):
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    one = Int4KvCache.allocate(1, 1, 32, 64, 32, device)
    desc = type(one.desc).from_buffer_copy(one.desc)
    desc.batch, desc.kv_heads, desc.capacity = rows, kv_heads, tokens          # (only asked for its size)
    need = backend.lib.tt_gqa_attention_int4_scratch_floats(desc, rows, heads, 0, 0, tokens)
    groups, tiles = rows * kv_heads * -(-(heads // kv_heads) // 16), -(-tokens // 32)
    if tiles <= 24 or (groups >= cus and tiles <= 64):
        splits = 1
    else:
        splits = max(min(max(1, 2 * cus // groups), -(-tiles // 8)), -(-tiles // 256))
    assert need == (0 if splits == 1 else rows * heads * splits * 66)
