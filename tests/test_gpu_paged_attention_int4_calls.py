"""Calls of the 4-bit cache's attention that a user may make of the prompt kernel as of the other one: queries that are not
finite, pages and lengths out of range, pages past 32 bits apart, results over the queries, captured calls and calls side by side;
steps under torch.compile; and the smallest and most numerous batches."""
from __future__ import annotations

import math

import pytest
import torch

import mas_b200
from mas_b200 import _lib
from parity import assert_bits_equal
from test_gpu_paged_attention_int4 import _cums, _make, _run, _takes_prompt_kernel

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
HQ, HKV, D = 32, 2, 128  # 16 rows a token and kv head


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prompt(seed, lens, qlens, dtype=BF, poison=False):
    """(q, cache, table, lens, cum): a call of which the requests with more than six queries go to the prompt kernel."""
    cache, table = _make(seed, lens, HKV, D, 16, "NHD", poison=poison)
    T = sum(qlens)
    assert any(_takes_prompt_kernel(T, len(lens), HQ, n * HQ // HKV) for n in qlens)
    q = torch.randn(T, HQ, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    return q, tuple(t.cuda() for t in cache), table.cuda(), _i32(lens), _i32(_cums(qlens))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_not_finite_queries_stay_in_their_prompt_rows(cuda, dtype):
    q, *args = _prompt(1, [500, 90], [300, 40], dtype)
    want = mas_b200.paged_attention_int4(q, *args)
    rows = [(0, 0, math.nan), (17, 31, math.inf), (150, 5, -math.inf), (299, 16, math.nan), (339, 3, math.nan)]
    for t, h, bad in rows:
        q[t, h, 7 * h % D] = bad
    got = mas_b200.paged_attention_int4(q, *args)
    for t, h, _ in rows:
        assert got[t, h].isnan().all()
        got[t, h] = want[t, h]
    assert_bits_equal(got, want, "other rows")


def test_pages_and_lengths_out_of_range_in_the_prompt_kernel(cuda):
    q, cache, table, lens, cum = _prompt(2, [500, 160], [300, 40])
    bad = table.clone()
    bad[0, 3], bad[0, 20], bad[1, 9] = cache[0].shape[0], -1, 1 << 30
    mas_b200.read_status(cuda)
    got = mas_b200.paged_attention_int4(q, cache, bad, lens, cum)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    # their tokens read as zeros: a page of zeros in their place gives the same bits
    more = tuple(torch.cat([t, torch.zeros_like(t[:1])]) for t in cache)
    same = table.clone()
    same[0, 3] = same[0, 20] = same[1, 9] = cache[0].shape[0]
    assert_bits_equal(got, mas_b200.paged_attention_int4(q, more, same, lens, cum), "bad pages read as zeros")
    assert mas_b200.read_status(cuda) == 0
    # lengths are cut to the table, a negative one to none
    full = table[:, :10].contiguous()
    want = mas_b200.paged_attention_int4(q, cache, full, _i32([160, 0]), cum)
    assert mas_b200.read_status(cuda) == 0
    got = mas_b200.paged_attention_int4(q, cache, full, _i32([1 << 30, -3]), cum)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    assert_bits_equal(got, want, "lengths cut")
    # query rows past the tensor are left out, rows that no request covers as they were
    out = torch.full_like(q, 9.0)
    mas_b200.paged_attention_int4(q, cache, table, lens, _i32([20, 400, 500]), out=out)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    want = mas_b200.paged_attention_int4(q, cache, table, lens, _i32([20, 340, 340]))
    assert (out[:20] == 9).all()
    assert_bits_equal(out[20:], want[20:], "queries cut")


def test_prompt_offsets_past_32_bits(cuda):
    """Pages 0.8 GB apart hold the same rows as a small cache."""
    far, n = 800_000_000, 80
    cache, table = _make(3, [n], HKV, D, 16, "NHD", poison=False)
    dev = tuple(t.cuda() for t in cache)
    pages = dev[0].shape[0]
    codes = []
    for t in dev[:2]:
        big = torch.empty((pages - 1) * far + t[0].numel(), dtype=torch.uint8, device=cuda)
        codes.append(big.as_strided(t.shape, (far, *t.stride()[1:])))
        codes[-1].copy_(t)
    q = torch.randn(320, HQ, D, device=cuda).to(BF)
    assert pages * far > 1 << 32 and _takes_prompt_kernel(320, 1, HQ, 320 * HQ // HKV)
    args = (table.cuda(), _i32([n]), _i32([0, 320]))
    want = mas_b200.paged_attention_int4(q, dev, *args, causal=False)
    got = mas_b200.paged_attention_int4(q, (codes[0], codes[1], dev[2]), *args, causal=False)
    assert_bits_equal(got, want, "far pages")


@pytest.mark.parametrize("lens,qlens", [([500, 700, 90, 3], [300, 1, 40, 2]), ([900, 4, 2000], [1, 2, 1]), ([6000], [320])])
def test_results_over_the_queries(cuda, lens, qlens):
    """out may be the query tensor itself: a row's queries are read by what writes the row alone."""
    cache, table = _make(4, lens, HKV, D, 16, "NHD")
    q = torch.randn(sum(qlens), HQ, D).to(BF).cuda()
    args = (tuple(t.cuda() for t in cache), table.cuda(), _i32(lens), _i32(_cums(qlens)))
    want = mas_b200.paged_attention_int4(q, *args)
    for _ in range(5):
        over = q.clone()
        assert mas_b200.paged_attention_int4(over, *args, out=over) is over
        assert_bits_equal(over, want, "in place")


def test_captured_prompt_steps_follow_the_lengths(cuda):
    """A captured step of prompt and decode rows, replayed with other lengths and queries, two graphs at once."""
    lens, qlens = [600, 900, 70, 300], [300, 1, 40, 3]
    cases = [_prompt(seed, lens, qlens) for seed in (5, 6)]
    cum = cases[0][4]
    cases = [(q, c, t, sl, cum) for q, c, t, sl, _ in cases]
    mas_b200.paged_attention_int4(*cases[0])
    graphs, outs = [], []
    for case in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mas_b200.paged_attention_int4(*case, return_lse=True))
        graphs.append(g)
    for now, new in (([600, 900, 70, 300], qlens), ([400, 800, 60, 300], [2, 1, 41, 300]), ([1, 1, 1, 1], [1, 1, 1, 1]),
                     ([344, 900, 0, 0], [344, 0, 0, 0])):
        cum.copy_(_i32(_cums(new)))
        for q, _, _, sl, _ in cases:
            sl.copy_(_i32(now))
            q.copy_(torch.randn(q.shape).to(BF))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for case, (out, lse) in zip(cases, outs):
            want, wlse = mas_b200.paged_attention_int4(*case, return_lse=True)
            assert_bits_equal(out[: sum(new)], want[: sum(new)], f"replay at {now}")
            assert_bits_equal(lse[: sum(new)], wlse[: sum(new)], f"lse at {now}")
    assert mas_b200.read_status(cuda) == 0 and mas_b200.read_fault_word(0) == 0


def test_prompt_calls_side_by_side(cuda):
    cases = [_prompt(seed, [700, 500], [320, 9]) for seed in range(7, 11)]
    want = [mas_b200.paged_attention_int4(*case) for case in cases]
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in cases]
    for s, case in zip(streams, cases):
        with torch.cuda.stream(s):
            for _ in range(3):
                out = mas_b200.paged_attention_int4(*case)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert_bits_equal(a, b, "streams side by side")
    assert mas_b200.read_fault_word(0) == 0


def test_more_requests_than_threads(cuda):
    _run(81, [40] * 600, [7] * 600, 16, 1, 64, BF)                            # all the prompt kernel's
    lens = [(7 * i) % 45 for i in range(1700)]
    qlens = [9 if i % 3 == 0 else i % 3 for i in range(1700)]
    _run(82, lens, qlens, 12, 1, 64, FP, page_size=5)                         # of both kernels


def test_nothing_to_see(cuda):
    """No tokens, no table columns, no queries, no requests."""
    cache = mas_b200.empty_paged_kv_cache_int4(2, 16, HKV, D)
    for T, cum in ((2, None), (2, [0, 1, 2]), (400, [0, 400, 400])):
        q = torch.randn(T, HQ, D, device=cuda).to(BF)
        for columns in (0, 1):
            table = torch.zeros(2, columns, dtype=torch.int32, device=cuda)
            out, lse = mas_b200.paged_attention_int4(q, cache, table, _i32([0, 0]), None if cum is None else _i32(cum), return_lse=True)
            assert (out == 0).all() and (lse == -math.inf).all()
    none = torch.empty(0, HQ, D, dtype=BF, device=cuda)
    table = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    assert mas_b200.paged_attention_int4(none, cache, table, _i32([0, 5]), _i32([0, 0, 0])).shape == none.shape
    assert mas_b200.paged_attention_int4(none, cache, table[:0], _i32([])).shape == none.shape
    assert mas_b200.read_status(cuda) == 0


def test_compiled_step(cuda):
    """A whole step under torch.compile, and the forms that write into given tensors: the same state and results as eager."""
    hq, hkv, d, batch, width = 8, 2, 64, 3, 4
    ptr = torch.arange(batch + 1, dtype=torch.int32, device=cuda) * width
    g = torch.Generator().manual_seed(9)
    new = _i32([5, 20, 1])
    q, k, v = (torch.randn(50, h, d, generator=g).to(BF).cuda() for h in (hq, hkv, hkv))

    def step(state, q, k, v, held):
        cache, sl, bt, fp, nf = state
        maps = mas_b200.allocate_paged_kv(new, sl, bt, fp, nf, 16, 50)
        flat = bt.flatten()
        mas_b200.append_paged_kv_cache_int4(k * 2, v, maps.batch_indices, maps.positions, cache, flat, ptr, maps.kv_last_page_len)
        out = mas_b200.paged_attention_int4(q, cache, bt, sl, maps.cum_append_lens, out=held[0])
        rows = mas_b200.read_paged_kv_cache_int4(maps.batch_indices, maps.positions, cache, flat, ptr)
        mas_b200.read_paged_kv_cache_int4(maps.batch_indices, maps.positions, cache, flat, ptr, out=(held[1], held[2]))
        mas_b200.release_paged_kv(sl - 1, sl, bt, fp, nf, 16)
        again = mas_b200.allocate_paged_kv(torch.ones_like(new), sl, bt, fp, nf, 16, 3, out=held[3])
        return out + 1, rows[0] + rows[1], again.positions + 1

    def fresh():
        state = (mas_b200.empty_paged_kv_cache_int4(12, 16, hkv, d), _i32([0, 3, 16]), _i32([[0] * 4, [11, 0, 0, 0], [10, 0, 0, 0]]),
                 torch.arange(12, dtype=torch.int32, device=cuda), _i32([10]))
        held = (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k),
                mas_b200.PagedKVMaps(_i32([0] * 4), _i32([0] * 3), _i32([0] * 3), _i32([0] * 3)))
        return state, held
    results = []
    for f in (step, torch.compile(step)):
        state, held = fresh()
        for _ in range(2):
            res = f(state, q, k, v, held)
        results.append([*res, *state[0], *state[1:], *held[:3], *held[3]])
    assert mas_b200.read_status(cuda) == 0
    for i, (a, b) in enumerate(zip(*results)):
        assert_bits_equal(b, a, f"compiled, {i}")
