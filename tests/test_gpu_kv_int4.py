"""The 4-bit append and read against exact rational arithmetic: codes, scales and minima bit for bit.

Rows that sit on borders (halves of a step, constants, denormals, the types' largest values), rows with NaN or
infinities, both layouts, page sizes of one and odd ones, strided and unaligned k/v, padding and out-of-range
tokens, caches whose offsets pass 32 bits. Values read back are c s + m rounded twice at most (fp32, then the
type): off by (eps / 2 + 2^-24) of the value.
"""
from __future__ import annotations

import math

import pytest
import torch

import kv_int4_ref as ref
import mas_b200
from mas_b200 import _lib, workloads
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _rows(seed, tokens, heads, d, dtype):
    """Rows of many kinds: plain, with outliers, offset, constant, on borders, tiny, huge."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, d, generator=g)
    kinds = torch.randint(0, 9, (tokens, heads), generator=g)
    kinds.view(-1)[:9] = torch.arange(9)[: kinds.numel()]
    for i in range(tokens):
        for h in range(heads):
            r, k = x[i, h], int(kinds[i, h])
            if k == 1:
                r *= 1 + 30 * (torch.rand(d, generator=g) < 0.05)
            elif k == 2:
                r += 100
            elif k == 3:
                r.fill_(float(r[0]))
            elif k == 4:  # integers and halves over a range of 15: exact ties
                r.copy_(torch.randint(0, 31, (d,), generator=g) / 2)
                r[0], r[1] = 0, 15
            elif k == 5:
                r *= 1e-39 if dtype == BF else 1e-7
            elif k == 6:
                big = 3.3e38 if dtype == BF else 6.5e4
                r.copy_(((torch.rand(d, generator=g) * 2 - 1).double() * big).float())
            elif k == 7:
                r.zero_()
                r[int(torch.randint(0, d, (1,), generator=g))] = -1.0
            elif k == 8:  # a few coarse values: many ties
                r.copy_(torch.randint(-6, 7, (d,), generator=g) * 0.375)
    return x.to(dtype)


def _check(k, v, cache, layout, b, dev_read, dtype):
    pos = b.positions.long()
    table = b.block_tables
    pages, entries = table[b.batch_indices.long(), pos // b.page_size].long(), pos % b.page_size
    kc, vc, pairs = (t.cpu() for t in cache)
    for which, (x, codes) in enumerate(((k, kc), (v, vc))):
        c = codes[pages, entries] if layout == "NHD" else codes[pages, :, entries]
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
        pr = pairs[pages, :, entries]
        for i in range(x.shape[0]):
            for h in range(x.shape[1]):
                want, s, m = ref.quantise_row(x[i, h])
                assert c[i, h].tolist() == want, (which, i, h)
                got = pr[i, h, 2 * which: 2 * which + 2].double().tolist()
                assert got == [s, m] or (math.isnan(s) and all(map(math.isnan, got))), (which, i, h, got, s, m)
    exact = ref.read_rows((kc, vc, pairs), layout, pages, entries)
    tol = torch.finfo(dtype).eps / 2 + 2.0 ** -24
    top = torch.finfo(dtype).max
    for got, want in zip(dev_read, exact):
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan())
        want = torch.where(want.isnan(), 0.0, want).clamp(-top, top)
        err = (torch.where(got.isnan(), 0.0, got) - want).abs()
        assert (err <= tol * want.abs() + 2.0 ** -134).all() if dtype == BF else (err <= tol * want.abs() + 2.0 ** -25).all()


def _append_and_check(seed, heads, d, dtype, layout, page_size, decodes, prompts, shape_rows=None, pdt=torch.int32):
    b = workloads.paged_batch(seed=seed, num_decodes=decodes, prompt_lens=prompts, page_size=page_size, max_cached=60)
    T = b.positions.shape[0]
    k, v = _rows(seed, T, heads, d, dtype), _rows(seed + 1, T, heads, d, dtype)
    cache = mas_b200.empty_paged_kv_cache_int4(b.num_pages, page_size, heads, d, layout)
    for t in cache[:2]:
        t.fill_(0xA5)
    cache[2].fill_(7.0)
    before = [t.clone() for t in cache]
    bd = b.to("cuda")
    kd, vd = (k.cuda(), v.cuda()) if shape_rows is None else shape_rows(k, v)
    mas_b200.read_status()
    mas_b200.append_paged_kv_cache_int4(kd, vd, bd.batch_indices, bd.positions.to(pdt), cache, bd.kv_indices, bd.kv_indptr,
                                        bd.kv_last_page_len, kv_layout=layout)
    got = mas_b200.read_paged_kv_cache_int4(bd.batch_indices, bd.positions.to(pdt), cache, bd.kv_indices, bd.kv_indptr,
                                            dtype=dtype, kv_layout=layout)
    assert mas_b200.read_status() == 0
    _check(k, v, cache, layout, b, got, dtype)
    # every other row of the cache is as it was
    pos = bd.positions.long()
    pages, entries = bd.block_tables[bd.batch_indices.long(), pos // page_size].long(), pos % page_size
    for t, old in zip(cache, before):
        if layout == "NHD" and t.dtype == torch.uint8:
            t[pages, entries] = old[pages, entries]
        else:
            t[pages, :, entries] = old[pages, :, entries]
        assert_bits_equal(t, old, "rows of other tokens")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads,d,layout,page_size,decodes,prompts", [
    (1, 128, "NHD", 16, 9, ()), (8, 128, "NHD", 16, 3, (9,)), (8, 128, "HND", 16, 3, (9,)), (3, 128, "HND", 5, 0, (11, 1)),
    (5, 64, "NHD", 1, 2, (5,)), (12, 64, "HND", 7, 1, (4,)), (16, 64, "NHD", 64, 2, (3,)), (17, 128, "NHD", 24, 1, (2,)),
])
def test_append_and_read(cuda, dtype, heads, d, layout, page_size, decodes, prompts):
    _append_and_check(heads + d, heads, d, dtype, layout, page_size, decodes, prompts)


def test_strided_views_of_a_qkv_row(cuda):
    def views(k, v):
        T, H, D = k.shape
        row = torch.full((T, 4 * D + 2 * H * D), 1e4, dtype=k.dtype)
        row[:, 4 * D: 4 * D + H * D] = k.reshape(T, -1)
        row[:, 4 * D + H * D:] = v.reshape(T, -1)
        row = row.cuda()
        return row[:, 4 * D: 4 * D + H * D].view(T, H, D), row[:, 4 * D + H * D:].view(T, H, D)
    _append_and_check(51, 4, 128, BF, "NHD", 16, 3, (6,), views, torch.int64)


@pytest.mark.parametrize("d", [64, 128])
def test_unaligned_rows(cuda, d):
    """Rows that start on odd elements with odd strides: the scalar loads."""
    def views(k, v):
        T, H, D = k.shape
        out = []
        for x in (k, v):
            buf = torch.full((T, H, D + 1), -1e4, dtype=k.dtype).cuda()
            buf[:, :, 1:] = x.cuda()
            out.append(buf[:, :, 1:])
        return out
    _append_and_check(52, 3, d, FP, "HND", 16, 3, (4,), views)


def test_read_into_unaligned_out(cuda):
    b = workloads.paged_batch(seed=3, num_decodes=5, prompt_lens=(7,), page_size=16).to(cuda)
    T = b.positions.shape[0]
    k, v = _rows(1, T, 3, 64, BF).cuda(), _rows(2, T, 3, 64, BF).cuda()
    cache = mas_b200.empty_paged_kv_cache_int4(b.num_pages, 16, 3, 64)
    mas_b200.append_paged_kv_cache_int4(k, v, b.batch_indices, b.positions, cache, b.kv_indices, b.kv_indptr, b.kv_last_page_len)
    plain = mas_b200.read_paged_kv_cache_int4(b.batch_indices, b.positions, cache, b.kv_indices, b.kv_indptr)
    buf = torch.full((2, T, 3, 67), 5.0, dtype=BF, device=cuda)
    out = (buf[0, :, :, 1:65], buf[1, :, :, 1:65])
    mas_b200.read_paged_kv_cache_int4(b.batch_indices, b.positions, cache, b.kv_indices, b.kv_indptr, out=out)
    for a, c in zip(out, plain):
        assert_bits_equal(a.contiguous(), c, "unaligned out")
    assert (buf[:, :, :, 0] == 5).all() and (buf[:, :, :, 65:] == 5).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_are_not_finite_read_as_nan(cuda, bad):
    T, H, D = 6, 2, 128
    k = torch.randn(T, H, D).to(BF)
    v = k.clone()
    k[1, 0, 5] = bad
    v[2, 1, D - 1] = bad
    v[3, 0, 0] = bad
    v[3, 0, 1] = -bad
    cache = mas_b200.empty_paged_kv_cache_int4(1, 16, H, D)
    z, pos = torch.zeros(T, dtype=torch.int32, device=cuda), torch.arange(T, dtype=torch.int32, device=cuda)
    tab, ptr, last = z[:1], torch.tensor([0, 1], dtype=torch.int32, device=cuda), torch.tensor([T], dtype=torch.int32, device=cuda)
    mas_b200.append_paged_kv_cache_int4(k.cuda(), v.cuda(), z, pos, cache, tab, ptr, last)
    kr, vr = mas_b200.read_paged_kv_cache_int4(z, pos, cache, tab, ptr)
    want_k, want_v = torch.zeros(T, H, dtype=torch.bool), torch.zeros(T, H, dtype=torch.bool)
    want_k[1, 0] = want_v[2, 1] = want_v[3, 0] = True
    assert torch.equal(kr.isnan().all(-1).cpu(), want_k) and torch.equal(kr.isnan().any(-1).cpu(), want_k)
    assert torch.equal(vr.isnan().all(-1).cpu(), want_v) and torch.equal(vr.isnan().any(-1).cpu(), want_v)


def test_padding_and_out_of_range_tokens(cuda):
    H, D, ps = 2, 64, 4
    k = torch.randn(7, H, D, device=cuda).to(BF)
    cache = mas_b200.empty_paged_kv_cache_int4(3, ps, H, D)
    table = torch.tensor([2, 0, 9, 1], dtype=torch.int32, device=cuda)   # two requests of two pages; 9 does not exist
    ptr = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda)
    last = torch.tensor([1, 1], dtype=torch.int32, device=cuda)

    def both(batch, pos):
        bi, p = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (batch, pos))
        n = len(batch)
        mas_b200.append_paged_kv_cache_int4(k[:n], k[:n], bi, p, cache, table, ptr, last)
        a = mas_b200.read_status(cuda)
        kr, _ = mas_b200.read_paged_kv_cache_int4(bi, p, cache, table, ptr)
        return a, mas_b200.read_status(cuda), kr
    a, r, kr = both([-1, -1], [0, 5])
    assert a == 0 and r == 0 and (kr == 0).all() and (cache[0] == 0).all() and (cache[2] == 0).all()
    for batch, pos in (([2], [0]), ([-2], [0]), ([0], [-1]), ([1], [8]), ([1], [0])):
        a, r, kr = both(batch, pos)
        assert a == _lib.STATUS_KV_SLOT_OUT_OF_RANGE and r == a, (batch, pos)
        assert (kr == 0).all() and (cache[0] == 0).all() and (cache[2] == 0).all()
    a, r, kr = both([0, -1, 7, 0, 1], [0, 0, 0, 7, 5])
    assert a == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    assert (kr[0] != 0).any() and (kr[3] != 0).any() and (kr[4] != 0).any() and (kr[1:3] == 0).all()


def test_offsets_past_32_bits(cuda):
    """Pages 1.2 GB apart: byte offsets beyond 2^31 and 2^32 hold the same rows as a small cache."""
    H, D, ps, far = 2, 128, 16, 1_200_000_000 // 16 * 16
    size = 4 * far + ps * H * D
    big = [torch.empty(size, dtype=torch.uint8, device=cuda) for _ in range(2)]
    codes = [t.as_strided((5, ps, H, D // 2), (far, H * D // 2, D // 2, 1)) for t in big]
    small = mas_b200.empty_paged_kv_cache_int4(5, ps, H, D)
    pairs = torch.zeros_like(small[2])
    n = 5 * ps
    k, v = (torch.randn(n, H, D, device=cuda).to(BF) for _ in range(2))
    bi, pos = torch.zeros(n, dtype=torch.int32, device=cuda), torch.arange(n, dtype=torch.int32, device=cuda)
    table = torch.tensor([4, 0, 3, 1, 2], dtype=torch.int32, device=cuda)
    ptr, last = torch.tensor([0, 5], dtype=torch.int32, device=cuda), torch.tensor([ps], dtype=torch.int32, device=cuda)
    res = []
    for cache in ((codes[0], codes[1], pairs), small):
        mas_b200.append_paged_kv_cache_int4(k, v, bi, pos, cache, table, ptr, last)
        q = torch.ones(1, 4, D, dtype=BF, device=cuda)
        res.append((*mas_b200.read_paged_kv_cache_int4(bi, pos, cache, table, ptr),
                    mas_b200.paged_attention_int4(q, cache, table[None], torch.tensor([n], dtype=torch.int32, device=cuda))))
    for a, b in zip(*res):
        assert_bits_equal(a, b, "far pages")


def test_other_stream_and_capture(cuda):
    b = workloads.paged_batch(seed=8, num_decodes=4, prompt_lens=(21,), page_size=16).to(cuda)
    T, H, D = b.positions.shape[0], 4, 128
    k, v = (torch.randn(T, H, D, device=cuda).to(BF) for _ in range(2))
    caches = [mas_b200.empty_paged_kv_cache_int4(b.num_pages, 16, H, D) for _ in range(3)]

    def step(cache):
        mas_b200.append_paged_kv_cache_int4(k, v, b.batch_indices, b.positions, cache, b.kv_indices, b.kv_indptr, b.kv_last_page_len)
        return mas_b200.read_paged_kv_cache_int4(b.batch_indices, b.positions, cache, b.kv_indices, b.kv_indptr)
    want = step(caches[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step(caches[1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step(caches[2])
    k.add_(0.5)
    graph.replay()
    changed = step(caches[0])
    torch.cuda.synchronize()
    for a, c in zip(want, other):
        assert_bits_equal(a, c, "another stream")
    for a, c in zip(changed, held):
        assert_bits_equal(a, c, "replay")
