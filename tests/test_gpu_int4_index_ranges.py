"""64-bit lengths and indices of the 4-bit cache's operators that int32 does not hold: refused or flagged as any other value out
of range, never taken for the value of their low 32 bits."""
from __future__ import annotations

import pytest
import torch

import mas_b200
from mas_b200 import _lib

pytestmark = pytest.mark.gpu

WIDE = [(1 << 32) + 1, (1 << 32), (1 << 31), -(1 << 32) + 1, -(1 << 32), (1 << 63) - 1, -(1 << 63)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("wide", WIDE)
@pytest.mark.parametrize("release", [False, True])
def test_page_lengths_past_32_bits_are_refused(cuda, wide, release):
    lens, free = [16, 40], [7, 8, 9, -2, -2, -2, -2]
    sl, bt, fp, nf = _i32(lens), _i32([[1, 0, 0, 0], [2, 3, 4, 0]]), _i32(free), _i32([3])
    delta = torch.tensor([1, wide], device="cuda")
    mas_b200.read_status(cuda)
    if release:
        mas_b200.release_paged_kv(delta, sl, bt, fp, nf, 16)
    else:
        maps = mas_b200.allocate_paged_kv(delta, sl, bt, fp, nf, 16, 8)
        assert set(maps.batch_indices.tolist()) == {-1}
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_ALLOC_REFUSED
    assert sl.tolist() == lens and nf.tolist() == [3] and fp.tolist() == free
    assert bt.tolist() == [[1, 0, 0, 0], [2, 3, 4, 0]]


@pytest.mark.parametrize("wide", WIDE + [(1 << 32) - 1])  # the last one's low half is the padding's -1
@pytest.mark.parametrize("which", ["batch_indices", "kv_indices", "kv_indptr"])
def test_slots_past_32_bits_are_flagged(cuda, wide, which):
    heads, dim = 2, 64
    cache = mas_b200.empty_paged_kv_cache_int4(3, 16, heads, dim)
    index = dict(batch_indices=[0, 1], kv_indices=[0, 2], kv_indptr=[0, 1, 2])
    index[which][1] = wide
    index = {name: torch.tensor(x, device="cuda") for name, x in index.items()}
    pos = _i32([3, 5])
    k = torch.randn(2, heads, dim, device="cuda").to(torch.bfloat16)
    mas_b200.read_status(cuda)
    mas_b200.append_paged_kv_cache_int4(k, k, index["batch_indices"], pos, cache, index["kv_indices"], index["kv_indptr"],
                                        _i32([4, 6]))
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    key, _ = mas_b200.read_paged_kv_cache_int4(index["batch_indices"], pos, cache, index["kv_indices"], index["kv_indptr"])
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    assert (key[0] != 0).any() and (key[1] == 0).all()
    written = (cache[2] != 0).any(-1).any(1)  # [pages, entries]
    assert written.nonzero().tolist() == [[0, 3]]
