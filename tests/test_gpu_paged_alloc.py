"""Page allocation and release on the GPU against a plain host block manager: exact.

Lengths of zero and one, pages of one and of odd sizes, requests that need no page, empty batches, one
cluster and one CTA, padded token maps, all-or-nothing refusals, in-place state carried by a captured graph, and
release as the inverse of allocation.
"""
from __future__ import annotations

import random

import pytest
import torch

import kv_int4_ref as ref
import mas_b200
from mas_b200 import _lib

pytestmark = pytest.mark.gpu


def _t(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _case(seed, batch, page_size, max_len, max_new, spare=5, extra_cols=1):
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, rng.randint(0, max_len)]) for _ in range(batch)]
    new = [rng.choice([0, 1, rng.randint(0, max_new)]) for _ in range(batch)]
    pages = lambda n: -(-n // page_size)  # noqa: E731
    width = max([pages(n + a) for n, a in zip(lens, new)] + [0]) + extra_cols
    used = sum(map(pages, lens))
    need = sum(pages(n + a) - pages(n) for n, a in zip(lens, new))
    pool = list(range(used + need + spare))
    rng.shuffle(pool)
    table = [[-7] * width for _ in range(batch)]
    for b, n in enumerate(lens):
        for j in range(pages(n)):
            table[b][j] = pool.pop()
    free = pool + [-3] * used  # capacity for every page
    return lens, new, table, free, len(pool), width


@pytest.mark.parametrize("seed,batch,page_size,max_len,max_new,pad", [
    (0, 1, 16, 40, 3, 0), (1, 7, 16, 300, 40, 5), (2, 33, 1, 50, 9, 1), (3, 256, 16, 4000, 1, 0),
    (4, 64, 5, 2000, 700, 100), (5, 1500, 24, 200, 30, 17), (6, 8192, 16, 30, 3, 3), (7, 3, 64, 5000, 20000, 0),
    (8, 1025, 7, 0, 11, 2),
])
def test_allocate_then_release(cuda, seed, batch, page_size, max_len, max_new, pad):
    lens, new, table, free, num_free, width = _case(seed, batch, page_size, max_len, max_new)
    max_tokens = sum(new) + pad
    sl, bt, fp, nf = _t(lens), _t(table), _t(free), _t([num_free])
    mas_b200.read_status(cuda)
    maps = mas_b200.allocate_paged_kv(_t(new), sl, bt, fp, nf, page_size, max_tokens)
    ok, cum, bi, pos, last, want_lens, want_table, want_free = ref.allocate(new, lens, table, free, num_free,
                                                                          page_size, max_tokens)
    assert ok and mas_b200.read_status(cuda) == 0
    assert maps.cum_append_lens.tolist() == cum
    assert maps.batch_indices.tolist() == bi and maps.positions.tolist() == pos
    assert maps.kv_last_page_len.tolist() == last
    assert sl.tolist() == want_lens and nf.tolist() == [want_free]
    assert bt.tolist() == want_table and fp.tolist() == free

    # part of it back (drafts rejected), then some requests finish
    rng = random.Random(seed + 1)
    keep = [n + rng.randint(0, a) for n, a in zip(lens, new)]
    for keep in (keep, [k if rng.random() < 0.5 else 0 for k in keep]):
        before = (sl.tolist(), fp.tolist(), int(nf))
        mas_b200.release_paged_kv(_t(keep), sl, bt, fp, nf, page_size)
        ok, want_lens, want_free_list, n = ref.release(keep, before[0], want_table, before[1], before[2], page_size)
        assert ok and mas_b200.read_status(cuda) == 0
        assert sl.tolist() == want_lens and nf.tolist() == [n] and fp.tolist() == want_free_list
        assert bt.tolist() == want_table


def test_release_restores_what_was_allocated(cuda):
    lens, new, table, free, num_free, _ = _case(11, 90, 16, 500, 60)
    sl, fp, nf, bt = _t(lens), _t(free), _t([num_free]), _t(table)
    mas_b200.allocate_paged_kv(_t(new).long(), sl, bt, fp, nf, 16, sum(new))
    mas_b200.release_paged_kv(_t(lens).long(), sl, bt, fp, nf, 16)
    assert sl.tolist() == lens and fp.tolist() == free and nf.tolist() == [num_free]


def test_empty_batch_and_no_new_tokens(cuda):
    sl, bt, fp, nf = _t([]), torch.empty((0, 4), dtype=torch.int32, device=cuda), _t([1, 2]), _t([2])
    maps = mas_b200.allocate_paged_kv(_t([]), sl, bt, fp, nf, 16, 3)
    assert maps.cum_append_lens.tolist() == [0] and maps.batch_indices.tolist() == [-1] * 3
    mas_b200.release_paged_kv(_t([]), sl, bt, fp, nf, 16)
    lens = [0, 5, 32]
    sl, bt = _t(lens), _t([[9, 9]] * 3)
    maps = mas_b200.allocate_paged_kv(_t([0, 0, 0]), sl, bt, fp, nf, 16, 0)
    assert maps.kv_last_page_len.tolist() == [0, 5, 16] and sl.tolist() == lens and nf.tolist() == [2]
    assert mas_b200.read_status(cuda) == 0


REFUSALS = [
    dict(new=[1, 40], free=2),             # too few free pages
    dict(new=[1, 200]),                    # past the table's columns
    dict(new=[-1, 1]),                     # negative
    dict(lens=[-5, 3]),
    dict(lens=[1 << 30, 3]),
    dict(new=[2, 2], max_tokens=3),        # more than the maps hold
    dict(new=[(1 << 31) - 1, (1 << 31) - 1]),
    dict(free=99),                         # a count past the list's end
    dict(free=-1),
]


@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("change", REFUSALS)
def test_allocate_refuses_whole(cuda, change, big):
    lens = change.get("lens", [16, 3])
    new = change.get("new", [1, 1])
    free = [10, 11, 12, 13, 14, 15, 16, 17]
    num = change.get("free", len(free))
    width = 6
    max_tokens = change.get("max_tokens", 60) + (5000 if big and "max_tokens" not in change else 0)
    sl, bt, fp, nf = _t(lens), _t([[4] * width, [5] * width]), _t(free), _t([num])
    mas_b200.read_status(cuda)
    maps = mas_b200.allocate_paged_kv(_t(new), sl, bt, fp, nf, 16, max_tokens)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_ALLOC_REFUSED
    assert sl.tolist() == lens and nf.tolist() == [num] and fp.tolist() == free
    assert bt.tolist() == [[4] * width, [5] * width]
    assert maps.cum_append_lens.tolist() == [0, 0, 0] and set(maps.batch_indices.tolist()) == {-1}
    assert maps.kv_last_page_len.tolist() == [(n - 1) % 16 + 1 if n > 0 else 0 for n in lens]


@pytest.mark.parametrize("keep,num", [([17, 0], 0), ([-1, 0], 0), ([0, 0], 4), ([0, 0], -1), ([0, 0], 9)])
def test_release_refuses_whole(cuda, keep, num):
    lens, free = [16, 40], [-2] * 7
    sl, bt, fp, nf = _t(lens), _t([[1, 0, 0], [2, 3, 4]]), _t(free), _t([num])
    mas_b200.read_status(cuda)
    mas_b200.release_paged_kv(_t(keep), sl, bt, fp, nf, 16)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_ALLOC_REFUSED
    assert sl.tolist() == lens and nf.tolist() == [num] and fp.tolist() == free


@pytest.mark.parametrize("batch,new", [(4, 3), (300, 20)])
def test_captured_steps_carry_the_state(cuda, batch, new):
    """Replays of one captured step continue where the last one stopped, and its out tensors are rewritten."""
    steps, page_size = 5, 16
    width = -(-steps * new // page_size)
    free = list(range(batch * width))
    state = dict(lens=[0] * batch, table=[[-1] * width for _ in range(batch)], num=len(free))
    sl, bt, fp, nf = _t(state["lens"]), _t(state["table"]), _t(free), _t([state["num"]])
    app = _t([new] * batch)
    maps = mas_b200.allocate_paged_kv(app, sl.clone(), bt.clone(), fp, nf.clone(), page_size, batch * new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mas_b200.allocate_paged_kv(app, sl, bt, fp, nf, page_size, batch * new, out=maps)
    for step in range(steps):
        now = [new if (b + step) % 3 else 0 for b in range(batch)]
        app.copy_(_t(now))
        graph.replay()
        ok, cum, bi, pos, last, lens, table, num = ref.allocate(now, state["lens"], state["table"], free, state["num"],
                                                              page_size, batch * new)
        assert ok
        assert maps.cum_append_lens.tolist() == cum and maps.batch_indices.tolist() == bi
        assert maps.positions.tolist() == pos and maps.kv_last_page_len.tolist() == last
        assert sl.tolist() == lens and bt.tolist() == table and nf.tolist() == [num]
        state = dict(lens=lens, table=table, num=num)
    assert mas_b200.read_status(cuda) == 0


def test_row_stride_of_the_table(cuda):
    """Block tables that are columns of a wider tensor: nothing outside them is written."""
    wide = _t([[50 + i for i in range(9)] for _ in range(4)])
    sl, fp, nf = _t([0, 3, 16, 31]), _t(list(range(100, 140))), _t([40])
    bt = wide[:, 2:6]
    mas_b200.allocate_paged_kv(_t([64, 20, 1, 1]), sl, bt, fp, nf, 16, 86)
    ok, *_, table, num = ref.allocate([64, 20, 1, 1], [0, 3, 16, 31], [[52, 53, 54, 55]] * 4, list(range(100, 140)), 40, 16, 86)
    assert ok and bt.tolist() == table and nf.tolist() == [num]
    assert wide[:, :2].tolist() == [[50, 51]] * 4 and wide[:, 6:].tolist() == [[56, 57, 58]] * 4
