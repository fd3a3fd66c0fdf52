"""Attention over the 4-bit cache against softmax(q k^T) v in 64 bits on the values the codes stand for.

Tolerance, per element, from the kernel's arithmetic (p normalised, n keys):
- a weight p s is rounded to fp16, 2^-11 of it and, with the largest near 1, not below 2^-25 of the largest; it multiplies the code
  c of 0..15 (bf16 results), c - 7.5 (fp16 ones) or c - 8 (the prompt kernel); the minima's part,
  sum p (m + z s) with z = 0, 7.5 or 8, has weights in fp32;
- sums over n keys in fp32, by steps of 16 in the matrix unit: u = 2^-22 (n / 16 + 32) of the terms' sizes;
- a logit is off by delta = sm_scale 2^-23 (D / 8 + 6) max_t (143 s_t + |m_t|) sum |q|: D / 16 steps of the matrix unit, two
  roundings each, and six more operations, on terms of at most 15 s |q|. It enters as 2 delta (sum p |v| + |o|);
- the result is rounded: eps_T / 2 |o|.
"""
from __future__ import annotations

import math
import os
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import kv_int4_ref as ref
import mas_b200
from mas_b200 import _lib
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _make(seed, lens, hkv, d, page_size, layout, poison=True, v_scale=1.0):
    """A cache with random codes and pairs like those of real rows, on the CPU; unused rows and pages hold NaN pairs."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page_size) for n in lens]
    width = max(blocks + [1]) + 1
    pages = sum(blocks) + 2
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), width), 0x7FFFFFF0, dtype=torch.int32)  # never to be looked up
    shape = (pages, page_size, hkv) if layout == "NHD" else (pages, hkv, page_size)
    codes = [torch.randint(0, 256, (*shape, d // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
    s = (0.2 + 0.3 * torch.rand(pages, hkv, page_size, 2, generator=g)) * torch.tensor([1.0, v_scale])
    m = -7.5 * s * (0.7 + 0.6 * torch.rand(pages, hkv, page_size, 2, generator=g))
    pairs = torch.stack([s, m], -1).flatten(-2).to(BF)
    o = 0
    keep = torch.zeros(pages, page_size, dtype=torch.bool)
    for b, (n, nb) in enumerate(zip(lens, blocks)):
        table[b, :nb] = perm[o:o + nb]
        for j in range(nb):
            keep[perm[o + j].long(), : min(page_size, n - j * page_size)] = True
        o += nb
    if poison:
        pairs = torch.where(keep[:, None, :, None], pairs, torch.tensor(math.nan, dtype=BF))
    return (codes[0], codes[1], pairs), table


def _takes_prompt_kernel(tokens: int, requests: int, hq: int, rows: int) -> bool:
    """The library's choice for a request with that many rows a kv head."""
    least = os.environ.get("MAS_ATTN_PROMPT_MIN_ROWS")
    least = int(least) if least else 64 * torch.cuda.get_device_properties(0).multi_processor_count
    return tokens > requests and rows > 96 and tokens * hq >= least


def _bound(q, cache, layout, table, lens, cum, scale, causal, dtype):
    """The 64-bit result, its lse, the tolerance, and the rows some request covers."""
    T, hq, d = q.shape
    ps, h = cache[2].shape[2], cache[2].shape[1]
    out, lse = ref.attention(q, cache, layout, table, lens, cum, scale, causal)
    tol = torch.zeros_like(out)
    ltol = torch.zeros_like(lse)
    for b, n in enumerate(lens):
        tok = torch.arange(n)
        pages, entries = table[b].long()[tok // ps], tok % ps
        k, v = ref.read_rows(cache, layout, pages, entries)
        pr = cache[2].double()[pages, :, entries]                       # [n, h, 4]
        # what the codes are centred on: the tensor-core kernel's rows, the other's for fp16 and for bf16
        z = 0.0 if dtype == BF else 7.5
        if _takes_prompt_kernel(T, len(lens), hq, (cum[b + 1] - cum[b]) * (hq // h)):
            z = 8.0
        code = (v - pr[..., 3, None]) / pr[..., 2, None]
        for i in range(cum[b], cum[b + 1]):
            seen = max(0, min(n, n - (cum[b + 1] - cum[b]) + (i - cum[b]) + 1)) if causal else n
            if seen == 0:
                continue
            qi = q[i].double().view(h, hq // h, d)
            p = torch.softmax(torch.einsum("hgd,thd->hgt", qi, k[:seen]) * scale, -1)
            steps = 2.0 ** -22 * (seen / 16 + 32)
            weights = torch.einsum("hgt,thd->hgd", p, (code[:seen] - z).abs() * pr[:seen, :, 2, None])
            weights = weights + 2.0 ** -14 * 15 * seen * (p * pr[:seen, :, 2].T[:, None]).amax(-1, keepdim=True)
            sums = torch.einsum("hgt,thd->hgd", p, code[:seen] * pr[:seen, :, 2, None])
            minima = torch.einsum("hgt,th->hg", p, (pr[:seen, :, 3].abs() + z * pr[:seen, :, 2]))[..., None]
            size = torch.einsum("hgt,thd->hgd", p, v[:seen].abs())
            reach = (143 * pr[:seen, :, 0] + pr[:seen, :, 1].abs()).amax(0)  # [h]
            delta = (2.0 ** -23 * (d / 8 + 6) * abs(scale) * reach[:, None] * qi.abs().sum(-1))[..., None]
            o = out[i].view(h, hq // h, d).abs()
            bound = 2.0 ** -11 * weights + steps * (sums + minima) + 2 * delta * (size + o) + torch.finfo(dtype).eps / 2 * o
            tol[i] = bound.reshape(hq, d) + torch.finfo(dtype).tiny
            # log2: the logits' error, the sum's and the logarithm's
            ltol[i] = (delta[..., 0] * 1.4427 + 2.0 ** -20 * (1 + lse[i].view(h, -1).abs())).reshape(hq) + steps
    return out, lse, tol, ltol


def _cums(qlens):
    cum = [0]
    for n in qlens:
        cum.append(cum[-1] + n)
    return cum


def _run(seed, lens, qlens, hq, hkv, d, dtype, page_size=16, layout="NHD", causal=True, scale=None, q_gain=1.0, tail=2,
         v_scale=1.0):
    cache, table = _make(seed, lens, hkv, d, page_size, layout, v_scale=v_scale)
    cum = _cums(qlens)
    T = cum[-1] + tail
    g = torch.Generator().manual_seed(seed + 1)
    # queries as a view of a wider row, results into a tensor whose other places are watched
    row = (torch.randn(T, hq * d + 40, generator=g) * q_gain).to(dtype)
    q = row[:, 40:].unflatten(-1, (hq, d))
    dev = [t.cuda() for t in cache]
    qd = row.cuda()[:, 40:].unflatten(-1, (hq, d))
    hold = torch.full((T, hq + 1, d + 8), 3.0, dtype=dtype, device="cuda")
    out = hold[:, :hq, :d]
    sl, cq = torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(cum, dtype=torch.int32).cuda()
    mas_b200.read_status()
    res, lse = mas_b200.paged_attention_int4(qd, tuple(dev), table.cuda(), sl, cq, sm_scale=scale, causal=causal,
                                             kv_layout=layout, out=out, return_lse=True)
    assert res is out and mas_b200.read_status() == 0
    again = mas_b200.paged_attention_int4(qd, tuple(dev), table.cuda(), sl, cq, sm_scale=scale, causal=causal, kv_layout=layout)
    assert_bits_equal(again[: cum[-1]], out[: cum[-1]], "run to run")
    assert (hold[cum[-1]:] == 3).all() and (hold[:, hq:] == 3).all() and (hold[:, :, d:] == 3).all()
    want, wlse, tol, ltol = _bound(q, cache, layout, table, lens, cum, d ** -0.5 if scale is None else scale, causal, dtype)
    n = cum[-1]
    err = (out[:n].cpu().double() - want[:n]).abs()
    assert not err.isnan().any()
    worst = (err / tol[:n].clamp(min=1e-300)).amax().item() if n else 0.0
    assert (err <= tol[:n]).all(), f"{worst} of the tolerance"
    empty = wlse[:n].isinf()
    assert torch.equal(lse[:n].cpu().isinf(), empty) and (out[:n].cpu()[empty] == 0).all()
    lerr = torch.where(empty, 0.0, (lse[:n].cpu().double() - torch.where(empty, 0.0, wlse[:n])).abs())
    assert (lerr <= ltol[:n]).all(), lerr.max()
    return worst


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (8, 2), (12, 1), (24, 8), (32, 2), (17, 1)])
def test_decode_heads(cuda, dtype, d, hq, hkv):
    lens = [1, 0, 2, 31, 32, 33, 127, 128, 129, 257, 600]
    _run(hq + d, lens, [1] * len(lens), hq, hkv, d, dtype)


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("page_size", [1, 5, 16, 24, 64, 256])
def test_page_sizes(cuda, layout, page_size):
    lens = [page_size, page_size + 1, max(1, page_size - 1), 3 * page_size + 2, 300]
    _run(page_size, lens, [1, 2, 1, 3, 5], 8, 2, 128, BF, page_size=page_size, layout=layout)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,qlens", [
    ([5, 40, 0, 300, 7], [3, 8, 2, 0, 7]),       # a request without tokens, one without queries, one all new
    ([3, 1], [9, 4]),                            # more queries than tokens: rows whose mask leaves nothing
    ([200, 129], [70, 129]),                     # many tiles
])
def test_ragged_queries(cuda, dtype, causal, lens, qlens):
    _run(7, lens, qlens, 12, 2, 64, dtype, causal=causal)
    _run(8, lens, qlens, 24, 2, 128, dtype, causal=causal, page_size=5, layout="HND")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,hq,hkv,lens,qlens", [
    (128, 12, 1, [50], [11]),                     # one step, two tiles of rows
    (128, 8, 1, [300], [10]),                     # one tile, several steps
    (64, 12, 2, [129, 128, 127], [30, 128, 7]),
    (128, 24, 2, [400, 3, 1000], [100, 3, 1]),    # beside short requests, which the other kernel takes
    (64, 4, 4, [0, 700, 90, 20], [0, 333, 90, 0]),
    (128, 17, 1, [40], [64]),                     # more queries than tokens
])
def test_prompt_rows(cuda, dtype, d, hq, hkv, lens, qlens):
    _run(61, lens, qlens, hq, hkv, d, dtype)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_rows_of_odd_pages_and_scales(cuda, causal):
    _run(62, [333, 70], [150, 70], 6, 2, 128, FP, page_size=5, layout="HND", causal=causal)
    _run(63, [333, 70], [150, 70], 6, 2, 128, BF, page_size=24, causal=causal, scale=-0.2)
    _run(64, [333], [150], 6, 2, 64, BF, page_size=1, causal=causal, q_gain=30.0)
    _run(65, [500], [40], 6, 2, 128, FP, causal=causal, v_scale=1e-4)
    _run(66, [500], [40], 6, 2, 128, BF, causal=causal, v_scale=1e30)


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_rows_of_a_long_context(cuda, causal):
    """One item of two tiles and one of a few rows, both cut into many parts."""
    _run(78, [6000, 5000], [40, 70], 4, 1, 128, BF, causal=causal)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_prompt_rows_beside_decode_rows(cuda, dtype):
    """A mixed step at the 123B-class head counts, large enough for the prompt kernel by itself."""
    _run(69, [450, 77, 300, 1, 130], [190, 1, 80, 1, 2], 96, 8, 128, dtype)


def test_small_prompts_through_the_prompt_kernel(cuda):
    """The prompt tests again in a process where the prompt kernel takes calls of any size."""
    env = dict(os.environ, MAS_ATTN_PROMPT_MIN_ROWS="0")
    here = Path(__file__).resolve()
    r = subprocess.run([sys.executable, "-m", "pytest", str(here), "-x", "-q", "-m", "gpu", "-k",
                        "prompt_rows or ragged or random_shapes or hidden_nan or decode_loop"], env=env, cwd=here.parents[1],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-2000:]


def test_prompt_rows_over_many_items_and_requests(cuda):
    rng = random.Random(5)
    lens = [rng.choice([0, 5, 200, 260]) for _ in range(70)]
    qlens = [min(n, rng.choice([0, 1, 40, 60])) for n in lens]
    _run(67, lens, qlens, 16, 4, 64, BF)


@pytest.mark.parametrize("seed", range(3))
def test_prompt_items_of_one_tile_before_items_of_two(cuda, seed):
    """Each CTA meets items of up to 128 rows, at many steps, between larger ones: the idle tile keeps its place."""
    rng = random.Random(70 + seed)
    qlens = [rng.choice([60, 64, 65, 100, 160, 200]) for _ in range(60)]  # 120 to 400 rows a kv head
    lens = [n + rng.choice([0, 130, 700, 1300]) for n in qlens]
    _run(71 + seed, lens, qlens, 16, 8, 64, BF)


@pytest.mark.parametrize("value", [-1.0, 1500.0, 1e9])
@pytest.mark.parametrize("tokens,new", [(2000, 1), (2000, 8), (2000, 1500)])
def test_constant_values(cuda, tokens, new, value):
    """Value rows without a spread have the smallest scale; the result is their minimum, whatever the weights are. Off by the
    result's rounding (2^-8) and the sums' (2^-22 (2000 / 16 + 32) < 2^-14)."""
    heads = 2
    cache = mas_b200.empty_paged_kv_cache_int4(tokens // 16 + 1, 16, heads, 128)
    table = torch.arange(tokens // 16 + 1, dtype=torch.int32, device="cuda")[None]
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(tokens, heads, 128, generator=g, device="cuda").to(BF)
    v = torch.full_like(k, value)
    mas_b200.append_paged_kv_cache_int4(k, v, torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                                        torch.arange(tokens, dtype=torch.int32, device="cuda"), cache, table.flatten(),
                                        torch.tensor([0, table.shape[1]], dtype=torch.int32, device="cuda"),
                                        torch.tensor([16], dtype=torch.int32, device="cuda"))
    q = torch.randn(new, 16, 128, generator=g, device="cuda").to(BF)
    out = mas_b200.paged_attention_int4(q, cache, table, torch.tensor([tokens], dtype=torch.int32, device="cuda"),
                                        torch.tensor([0, new], dtype=torch.int32, device="cuda"))
    want = v[0, 0, 0].double()
    assert ((out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -14) * want.abs()).all()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current(cuda):
    """One step's operators on cuda:1 while cuda:0 is current."""
    dev = torch.device("cuda:1")
    lens, qlens = [70, 5], [1, 2]
    cache, table = _make(77, lens, 2, 128, 16, "NHD")
    q = torch.randn(3, 8, 128).to(BF)
    i32 = dict(dtype=torch.int32)
    args = (table, torch.tensor(lens, **i32), torch.tensor([0, 1, 3], **i32))
    want = mas_b200.paged_attention_int4(q.cuda(0), tuple(t.cuda(0) for t in cache), *[t.cuda(0) for t in args])
    got = mas_b200.paged_attention_int4(q.to(dev), tuple(t.to(dev) for t in cache), *[t.to(dev) for t in args])
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(dev)
    assert_bits_equal(got.cpu(), want.cpu(), "cuda:1")


def test_hidden_nan_keys_do_not_reach_earlier_prompt_rows(cuda):
    lens, qlens = [150], [100]
    cache, table = _make(68, lens, 2, 128, 16, "NHD")
    q = torch.randn(100, 8, 128).to(BF).cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor([0, 100], dtype=torch.int32).cuda())
    want = mas_b200.paged_attention_int4(q, tuple(t.cuda() for t in cache), *args)
    for column in (slice(0, 2), slice(2, 4)):  # the keys' pair, the values' pair
        bad = [t.clone() for t in cache]
        t = 120  # seen by queries 70 and on
        bad[2][table[0, t // 16].long(), :, t % 16, column] = math.nan
        got = mas_b200.paged_attention_int4(q, tuple(t.cuda() for t in bad), *args)
        assert_bits_equal(got[:70], want[:70], "queries before the NaN")
        assert got[70:].isnan().all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_long_contexts_are_split_and_joined(cuda, dtype):
    _run(21, [20011], [1], 12, 1, 128, dtype)
    _run(22, [6000, 1, 9001], [2, 1, 3], 4, 1, 64, dtype, page_size=64, layout="HND")


def test_sharp_and_flat_softmax(cuda):
    _run(31, [700, 64], [1, 4], 8, 2, 128, BF, q_gain=30.0)     # logits of hundreds: one key takes all
    _run(32, [700, 64], [1, 4], 8, 2, 128, BF, q_gain=0.0)      # all keys alike
    _run(33, [700, 64], [1, 4], 8, 2, 128, FP, scale=-0.3)
    _run(34, [300], [1], 8, 2, 128, FP, v_scale=1e-4)           # small values keep their relative precision
    _run(35, [300], [1], 8, 2, 128, BF, v_scale=1e30)


def test_random_shapes(cuda):
    for seed in range(12):
        rng = random.Random(seed)
        hkv = rng.choice([1, 2, 3, 8])
        batch = rng.randint(1, 9)
        lens = [rng.choice([0, 1, rng.randint(1, 700)]) for _ in range(batch)]
        qlens = [rng.choice([0, 1, 1, 1, rng.randint(2, 30)]) for _ in range(batch)]
        _run(100 + seed, lens, qlens, hkv * rng.randint(1, 20), hkv, rng.choice([64, 128]), rng.choice([BF, FP]),
             page_size=rng.choice([1, 3, 8, 16, 100]), layout=rng.choice(["NHD", "HND"]), causal=rng.random() < 0.7)


def test_hidden_nan_keys_do_not_reach_earlier_queries(cuda):
    """Key and value rows of NaN belong to the newest tokens: the queries before them give what they gave without."""
    lens, qlens, d = [80, 40], [4, 3], 128
    cache, table = _make(41, lens, 2, d, 16, "NHD")
    q = torch.randn(7, 8, d).to(BF).cuda()
    args = (table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor([0, 4, 7], dtype=torch.int32).cuda())
    want = mas_b200.paged_attention_int4(q, tuple(t.cuda() for t in cache), *args)
    bad = [t.clone() for t in cache]
    for b, n in enumerate(lens):
        t = n - 2  # the last two tokens: visible to the last two queries and to the last one
        bad[2][table[b, t // 16].long(), :, t % 16] = math.nan
    got = mas_b200.paged_attention_int4(q, tuple(t.cuda() for t in bad), *args)
    assert_bits_equal(got[[0, 1, 4]], want[[0, 1, 4]], "queries before the NaN")
    assert got[[2, 3, 5, 6]].isnan().all()


def test_not_finite_queries_stay_in_their_rows(cuda):
    cache, table = _make(42, [50, 60], 2, 64, 16, "NHD")
    q = torch.randn(2, 8, 64).to(BF).cuda()
    args = (tuple(t.cuda() for t in cache), table.cuda(), torch.tensor([50, 60], dtype=torch.int32).cuda())
    want = mas_b200.paged_attention_int4(q, *args)
    q[0, 3, 7] = math.nan
    q[1, 6, 0] = math.inf
    got = mas_b200.paged_attention_int4(q, *args)
    assert got[0, 3].isnan().all() and got[1, 6].isnan().all()
    got[0, 3] = want[0, 3]
    got[1, 6] = want[1, 6]
    assert_bits_equal(got, want, "other rows")


def test_pages_and_lengths_out_of_range(cuda):
    d, ps = 128, 16
    cache, table = _make(43, [40, 40], 1, d, ps, "NHD", poison=False)
    q = torch.randn(2, 4, d).to(BF)
    dev = tuple(t.cuda() for t in cache)
    sl = torch.tensor([40, 40], dtype=torch.int32).cuda()
    bad = table.clone()
    bad[1, 1] = cache[0].shape[0]
    bad[0, 2] = -1
    mas_b200.read_status(cuda)
    got = mas_b200.paged_attention_int4(q.cuda(), dev, bad.cuda(), sl)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    # their tokens read as zeros: a page of zeros in their place gives the same bits
    zero = [torch.cat([t, torch.zeros_like(t[:1])]) for t in cache]
    same = table.clone()
    same[1, 1] = same[0, 2] = cache[0].shape[0]
    want = mas_b200.paged_attention_int4(q.cuda(), tuple(t.cuda() for t in zero), same.cuda(), sl)
    assert mas_b200.read_status(cuda) == 0
    assert_bits_equal(got, want, "bad pages read as zeros")
    # lengths are cut to the table (3 pages used, 4 columns with the last one bad) and to the queries
    full = table[:, :3].contiguous().cuda()
    want = mas_b200.paged_attention_int4(q.cuda(), dev, full, torch.tensor([48, 0], dtype=torch.int32).cuda())
    mas_b200.read_status(cuda)
    got = mas_b200.paged_attention_int4(q.cuda(), dev, full, torch.tensor([1 << 30, -3], dtype=torch.int32).cuda())
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    assert_bits_equal(got, want, "lengths cut")
    out = torch.full_like(q, 9.0).cuda()
    mas_b200.paged_attention_int4(q.cuda(), dev, full, sl, torch.tensor([1, 5, 4], dtype=torch.int32).cuda(), out=out)
    assert mas_b200.read_status(cuda) == _lib.STATUS_KV_SLOT_OUT_OF_RANGE
    assert (out[0] == 9).all()


def test_captured_call_follows_the_lengths(cuda):
    """One captured call, replayed with other lengths, queries and cached values; a second graph beside it."""
    d, hq, hkv = 128, 24, 2
    lens = [700, 3, 128, 1500]
    cache, table = _make(51, lens, hkv, d, 16, "NHD", poison=False)
    dev = tuple(t.cuda() for t in cache)
    tab = table.cuda()
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    qs = [torch.randn(4, hq, d).to(BF).cuda() for _ in range(2)]
    mas_b200.paged_attention_int4(qs[0], dev, tab, sl)
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mas_b200.paged_attention_int4(q, dev, tab, sl))
        graphs.append(g)
    for now in ([700, 3, 128, 1500], [1, 0, 100, 1400], [512, 2, 64, 130]):
        sl.copy_(torch.tensor(now, dtype=torch.int32))
        for q in qs:
            q.copy_(torch.randn(4, hq, d).to(BF))
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for q, o in zip(qs, outs):
            assert_bits_equal(o, mas_b200.paged_attention_int4(q, dev, tab, sl), f"replay at {now}")


def test_two_calls_at_once(cuda):
    cache, table = _make(52, [3000, 2000], 2, 128, 16, "NHD", poison=False)
    dev, tab, sl = tuple(t.cuda() for t in cache), table.cuda(), torch.tensor([3000, 2000], dtype=torch.int32).cuda()
    qs = [torch.randn(2, 24, 128).to(BF).cuda() for _ in range(4)]
    want = [mas_b200.paged_attention_int4(q, dev, tab, sl) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for s, q in zip(streams, qs):
        with torch.cuda.stream(s):
            for _ in range(3):
                r = mas_b200.paged_attention_int4(q, dev, tab, sl)
            got.append(r)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert_bits_equal(a, b, "streams side by side")


def test_compiled_call(cuda):
    cache, table = _make(53, [90, 20], 2, 64, 16, "NHD", poison=False)
    dev, tab, sl = tuple(t.cuda() for t in cache), table.cuda(), torch.tensor([90, 20], dtype=torch.int32).cuda()
    q = torch.randn(2, 8, 64).to(BF).cuda()

    def f(q, sl):
        return mas_b200.paged_attention_int4(q, dev, tab, sl) + 1
    assert_bits_equal(torch.compile(f, dynamic=True)(q, sl), f(q, sl), "compiled")


def test_a_decode_loop_of_all_operators(cuda):
    """Requests of ragged prompts, then steps with drafts of which some are rejected: pages from the GPU, rope, the 4-bit
    append, attention, release; against the same loop in plain form over the values the cache stands for."""
    hq, hkv, d, ps, dtype = 12, 2, 128, 16, BF
    prompts = [37, 1, 64, 90]
    batch, width = len(prompts), 16
    pool = batch * width
    cache = mas_b200.empty_paged_kv_cache_int4(pool, ps, hkv, d)
    table = torch.zeros(batch, width, dtype=torch.int32, device=cuda)
    free, num = torch.randperm(pool).to(torch.int32).cuda(), torch.tensor([pool], dtype=torch.int32, device=cuda)
    sl = torch.zeros(batch, dtype=torch.int32, device=cuda)
    ptr = torch.arange(batch + 1, dtype=torch.int32, device=cuda) * width
    rope = mas_b200.plain_cos_sin_cache(d, 512, 1e4).cuda()
    g = torch.Generator().manual_seed(3)
    rng = random.Random(3)
    held = [[] for _ in range(batch)]  # each request's (k, v) rows in 64 bits
    for step in range(5):
        new = prompts if step == 0 else [rng.randint(0, 5) for _ in range(batch)]
        T = sum(new)
        qkv = torch.randn(T + 3, (hq + 2 * hkv) * d, generator=g).to(dtype).cuda()  # three padding rows
        maps = mas_b200.allocate_paged_kv(torch.tensor(new, dtype=torch.int32, device=cuda), sl, table, free, num, ps, T + 3)
        q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=-1)
        mas_b200.apply_rope_with_cos_sin_cache_inplace(maps.positions, q, k, d, rope)
        mas_b200.append_paged_kv_cache_int4(k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d)), maps.batch_indices,
                                            maps.positions, cache, table.flatten(), ptr, maps.kv_last_page_len)
        got = mas_b200.paged_attention_int4(q, cache, table, sl, maps.cum_append_lens)
        assert mas_b200.read_status(cuda) == 0
        lens = [len(h) + n for h, n in zip(held, new)]
        assert sl.tolist() == lens
        cum = _cums(new)
        kf, vf = (x.reshape(-1, hkv, d).cpu() for x in (k, v))
        for b in range(batch):
            for i in range(cum[b], cum[b + 1]):
                rows = []
                for x in (kf, vf):
                    rows.append([(ref.quantise_row(x[i, h])) for h in range(hkv)])
                held[b].append(tuple(torch.stack([torch.tensor(c, dtype=torch.float64) * s + m for c, s, m in r]) for r in rows))
        # the cache holds exactly these rows ...
        host = tuple(t.cpu() for t in cache)
        tab = table.cpu()
        for b in range(batch):
            if lens[b]:
                tok = torch.arange(lens[b])
                hk, hv = ref.read_rows(host, "NHD", tab[b].long()[tok // ps], tok % ps)
                assert torch.equal(hk, torch.stack([r[0] for r in held[b]])) and torch.equal(hv, torch.stack([r[1] for r in held[b]]))
        # ... and attention is theirs
        qh = q.reshape(-1, hq, d).cpu()
        want, _, tol, _ = _bound(qh, host, "NHD", tab, lens, cum, d ** -0.5, True, dtype)
        err = (got.view(-1, hq, d)[:T].cpu().double() - want[:T]).abs()
        assert (err <= tol[:T]).all()
        keep = [n - (rng.randint(0, a) if step else 0) for n, a in zip(lens, new)]
        if step == 3:
            keep[2] = 0  # a request ends
        mas_b200.release_paged_kv(torch.tensor(keep, dtype=torch.int32, device=cuda), sl, table, free, num, ps)
        held = [h[:n] for h, n in zip(held, keep)]
        assert int(num) == pool - sum(-(-n // ps) for n in keep)
    assert mas_b200.read_status(cuda) == 0
