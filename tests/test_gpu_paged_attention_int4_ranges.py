"""Attention over the 4-bit cache at the ends of its ranges: value and key rows of very unlike scales in one cache, constant
rows, logits far apart, small queries under a large scale.

All requests of a call have the same lengths here, so the 64-bit form is a few dense products. Tolerance, per element, with p
normalised over n keys, w = p s the weight that a key's code carries, z what the codes are centred on (0: bf16 results, 7.5: fp16
ones, 8: the prompt kernel):
- w is rounded to fp16: 2^-11 of it (twice in the prompt kernel, where the reference may move between the halves of a step), and,
  below fp16's normal numbers, half of their step 2^-24 or all of w. The largest weight since its reference last moved lies in 1/2 to
  1024: the step is at most 2^-23 of the row's largest w. In the prompt kernel the reference follows the largest of
  max(s, |m + 8 s| 2^-60, 2^-96) p, up to a spread of 2^10 within a step, from below 2^8: 2^-14 of the largest such product;
- sums over n keys in fp32, by steps of 16 in the matrix unit: u = 2^-22 (n / 16 + 32) of the terms' sizes, at most (15 + z) w and
  p (|m| + z s);
- a logit is off by delta = sm_scale 2^-23 (D / 8 + 6) max_t (143 s_t + |m_t|) sum |q| (of the keys): D / 16 steps of the matrix unit,
  two roundings each, and six more operations, on terms of at most 15 s |q|. It enters as 2 delta (sum p |v| + |o|);
- a p below 2^-126 of its reference, which is at most 2^20 from the largest, is zero: 2^-100 of the largest |v|, n times; a
  weight below all the types' ranges: 16 steps of 2^-126;
- the result is rounded: eps_T / 2 |o|, or half a step of fp16's least numbers.
"""
from __future__ import annotations

import math
import os

import pytest
import torch

import mas_b200

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
LEAST = 2.0 ** -126  # a constant row's scale


def _prompt_kernel(tokens: int, requests: int, hq: int, rows: int) -> bool:
    """The library's choice for requests with that many rows a kv head."""
    least = os.environ.get("MAS_ATTN_PROMPT_MIN_ROWS")
    least = int(least) if least else 64 * torch.cuda.get_device_properties(0).multi_processor_count
    return tokens > requests and rows > 96 and tokens * hq >= least


def _cache(codes, kp, vp, page_size, layout):
    """A paged cache with the given rows, pages in a shuffled order. codes: two [B, n, h, D] of 0..15; kp, vp: [B, n, h, 2]."""
    B, n, h, d = codes[0].shape
    blocks = -(-n // page_size)
    table = torch.randperm(B * blocks, device="cuda").to(torch.int32).view(B, blocks)
    cache = mas_b200.empty_paged_kv_cache_int4(B * blocks, page_size, h, d, layout)
    cache[2].fill_(math.nan)
    tok = torch.arange(n, device="cuda")
    pages, entries = table[:, tok // page_size].long(), (tok % page_size).expand(B, n)
    for t, c in zip(cache, codes):
        packed = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
        if layout == "NHD":
            t[pages, entries] = packed
        else:
            t[pages, :, entries] = packed
    cache[2][pages, :, entries] = torch.cat([kp, vp], -1)
    return cache, table


def _codes(g, shape):
    return torch.randint(0, 16, shape, generator=g, device="cuda")


def _expect(q, codes, kp, vp, ql, scale, causal, prompt):
    """(out, tol, lse, ltol): [B * ql, hq, D], lse [B * ql, hq], in 64 bits."""
    B, n, h, d = codes[0].shape
    hq = q.shape[1]
    dtype = q.dtype
    kc, vc, kp, vp = codes[0].double(), codes[1].double(), kp.double(), vp.double()
    k, v = (c * p[..., :1] + p[..., 1:] for c, p in ((kc, kp), (vc, vp)))
    qd = q.double().view(B, ql, h, hq // h, d)
    s = torch.einsum("bqhgd,bnhd->bhgqn", qd, k) * scale
    if causal:
        seen = torch.arange(n, device="cuda") <= torch.arange(n - ql, n, device="cuda")[:, None]
        s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None].isinf(), 0.0, (s - lse[..., None]).exp())
    mix = lambda w, x: torch.einsum("bhgqn,bnhd->bhgqd", w, x)  # noqa: E731
    out = mix(p, v)
    z = 8.0 if prompt else 7.5 if dtype == FP else 0.0
    col = lambda x: x.transpose(1, 2)[:, :, None, None]  # noqa: E731  [b, n, h] -> [b, h, 1, 1, n]
    sv, mv = col(vp[..., 0]), col(vp[..., 1])
    w = p * sv
    if prompt:
        reach = torch.maximum(torch.maximum(sv, (mv + 8 * sv).abs() * 2.0 ** -60), torch.tensor(2.0 ** -96, device="cuda"))
        least = 2.0 ** -14 * (p * reach).amax(-1, keepdim=True)
    else:
        least = 2.0 ** -23 * w.amax(-1, keepdim=True)
    err = mix((2.0 ** -10 if prompt else 2.0 ** -11) * w + torch.minimum(w, least), (vc - z).abs())
    u = 2.0 ** -22 * (n / 16 + 32)
    err = err + u * (w * (15 + z) + p * (mv.abs() + z * sv)).sum(-1, keepdim=True)
    keys = (143 * kp[..., 0] + kp[..., 1].abs()).amax(1)  # [b, h]
    delta = 2.0 ** -23 * (d / 8 + 6) * abs(scale) * keys[:, :, None, None] * qd.abs().sum(-1).permute(0, 2, 3, 1)
    err = err + 2 * delta[..., None] * (mix(p, v.abs()) + out.abs())
    largest = torch.where(s.isinf(), 0.0, col(v.abs().amax(-1))).amax(-1, keepdim=True)
    err = err + n * 2.0 ** -100 * largest + 16 * LEAST
    err = err + torch.finfo(dtype).eps / 2 * torch.maximum(out.abs(), torch.tensor(torch.finfo(dtype).tiny, device="cuda"))
    lse2 = lse / math.log(2)
    ltol = delta * 1.4427 + 2.0 ** -20 * (1 + lse2.abs()) + u
    back = lambda x: x.permute(0, 3, 1, 2, *range(4, x.dim())).reshape(B * ql, hq, *x.shape[4:])  # noqa: E731
    return back(out), back(err), back(lse2), back(ltol)


def _check(q, codes, kp, vp, ql, dtype, scale=None, causal=True, layout="NHD", page_size=16):
    B, n, h, d = codes[0].shape
    q = q.to(dtype)
    scale = d ** -0.5 if scale is None else scale
    cache, table = _cache(codes, kp, vp, page_size, layout)
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    cum = torch.arange(B + 1, dtype=torch.int32, device="cuda") * ql
    mas_b200.read_status()
    got, glse = mas_b200.paged_attention_int4(q, cache, table, lens, cum, sm_scale=scale, causal=causal, kv_layout=layout,
                                              return_lse=True)
    assert mas_b200.read_status() == 0
    prompt = _prompt_kernel(B * ql, B, q.shape[1], ql * q.shape[1] // h)
    want, tol, lse, ltol = _expect(q, codes, kp, vp, ql, scale, causal, prompt)
    top = torch.finfo(dtype).max
    assert want.abs().max() < top
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), tol[bad][0].item())
    hidden = lse.isinf()
    assert torch.equal(glse.isinf(), hidden) and (got[hidden] == 0).all()
    lerr = torch.where(hidden, 0.0, (glse.double() - torch.where(hidden, 0.0, lse)).abs())
    assert (lerr <= ltol).all(), lerr.max()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pairs(s, m):
    return torch.stack([s, m], -1).to(BF)


def _plain_pairs(g, shape, scale=1.0):
    s = (0.2 + 0.3 * torch.rand(shape, generator=g, device="cuda")) * scale
    return _pairs(s, -7.5 * s * (0.7 + 0.6 * torch.rand(shape, generator=g, device="cuda")))


def _given_logits(logits):
    """Constant key rows of 128 or 64 elements that meet queries of ones, at scale 1 / D, in these logits."""
    return _pairs(torch.full_like(logits, LEAST), logits)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("group,ql", [(4, 1), (12, 1), (4, 8)])
@pytest.mark.parametrize("logit,value", [(70.0, 2.0 ** 40), (87.0, 2.0 ** 22), (87.0, -3.0), (300.0, 2.0 ** 15), (9.0, 2.0 ** 88)])
def test_a_constant_value_far_above_the_logits_before_it(cuda, dtype, group, ql, logit, value):
    """A value row without a spread weighs next to nothing, however large its p is; its minimum counts with that p."""
    if dtype == FP and abs(value) > 60000:
        value = math.copysign(60000.0, value)
    B, n, d = 500, 288, 128
    g = _gen(1)
    codes = [_codes(g, (B, n, 1, d)) for _ in range(2)]
    logits = torch.rand(B, n, 1, generator=g, device="cuda") * 2 - 1
    vp = _plain_pairs(g, (B, n, 1))
    at = 128 + torch.arange(B, device="cuda") % 120  # in the second run of a warp or later
    rows = torch.arange(B, device="cuda")
    logits[rows, at] = logit
    codes[0].zero_()
    codes[1][rows, at] = 0
    vp[rows, at, 0] = torch.tensor([LEAST, value], device="cuda").to(BF)
    q = torch.ones(B * ql, group, d, device="cuda")
    _check(q, codes, _given_logits(logits), vp, ql, dtype, scale=1 / d)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("first", ["constant", "zero pair"])
@pytest.mark.parametrize("wide", [2.0, 8.0, 2000.0])
@pytest.mark.parametrize("ql", [2, 8])
def test_a_hidden_wide_row_after_constant_ones(cuda, dtype, first, wide, ql):
    """Draft j sees the constant rows alone, as the newest token's wide value row is hidden from all but the last."""
    d, n = 128, ql
    codes = [torch.zeros(1, n, 2, d, dtype=torch.int64, device="cuda") for _ in range(2)]
    codes[1][0, -1] = _codes(_gen(2), (2, d))
    kp = _plain_pairs(_gen(3), (1, n, 2))
    vp = torch.zeros(1, n, 2, 2, dtype=BF, device="cuda")
    vp[..., 0], vp[..., 1] = (LEAST, 1.5) if first == "constant" else (0.0, 0.0)
    vp[0, -1] = torch.tensor([wide, -7.5 * wide], device="cuda").to(BF)
    q = torch.randn(ql, 8, d, generator=_gen(4), device="cuda")
    for causal in (True, False):
        _check(q, codes, kp, vp, ql, dtype, causal=causal)
    cache, table = _cache(codes, kp, vp, 16, "NHD")
    out = mas_b200.paged_attention_int4(q.to(dtype), cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                        torch.tensor([0, ql], dtype=torch.int32, device="cuda"))
    assert (out[0] == vp[0, 0, 0, 1]).all()  # one key: its minimum, which the type holds


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gap", [60.0, 88.0, 200.0])
def test_a_wide_row_far_below_constant_ones(cuda, dtype, gap):
    """Wide value rows whose p is next to nothing, or flushed to zero, beside attended constant rows of the same step."""
    B, n, d = 40, 96, 128
    g = _gen(5)
    codes = [_codes(g, (B, n, 2, d)) for _ in range(2)]
    logits = torch.rand(B, n, 2, generator=g, device="cuda")
    far = torch.rand(B, n, 2, generator=g, device="cuda") < 0.3
    logits = torch.where(far, logits - gap, logits)
    codes[0].zero_()
    vp = _plain_pairs(g, (B, n, 2), 500.0)
    vp = torch.where(far[..., None], vp, torch.tensor([LEAST, -2.0], device="cuda").to(BF))
    codes[1][~far] = 0
    _check(torch.ones(B, 8, d, device="cuda"), codes, _given_logits(logits), vp, 1, dtype, scale=1 / d)


@pytest.mark.parametrize("top", [30.0, 95.0])
def test_a_constant_row_above_the_widest(cuda, top):
    """Rows of scales near 2^95 first, then a constant row far above them: the sums are scaled down by less than fp32 holds."""
    B, n, d = 500, 288, 128
    g = _gen(6)
    codes = [_codes(g, (B, n, 1, d)) for _ in range(2)]
    logits = torch.rand(B, n, 1, generator=g, device="cuda")
    vp = _plain_pairs(g, (B, n, 1), 2.0 ** 85)
    at, rows = 128 + torch.arange(B, device="cuda") % 120, torch.arange(B, device="cuda")
    logits[rows, at] = top
    codes[0].zero_()
    codes[1][rows, at] = 0
    vp[rows, at, 0] = torch.tensor([LEAST, 2.0 ** 80], device="cuda").to(BF)
    _check(torch.ones(B, 4, d, device="cuda"), codes, _given_logits(logits), vp, 1, BF, scale=1 / d)


def _mixed_pairs(g, order, B, n, h, top):
    """Value rows of scales 2^-30 to 2^top over a cache, a tenth of them constant, a tenth without a pair."""
    e = torch.linspace(-30, top, n, device="cuda")[None, :, None] + torch.rand(B, n, h, generator=g, device="cuda")
    if order == "falling":
        e = e.flip(1)
    elif order == "shuffled":
        e = e[:, torch.randperm(n, generator=g, device="cuda")]
    s = torch.exp2(e)
    m = -7.5 * s * (0.7 + 0.6 * torch.rand(B, n, h, generator=g, device="cuda"))
    kind = torch.rand(B, n, h, generator=g, device="cuda")
    if order == "halves":
        kind = torch.where(torch.arange(n, device="cuda")[:, None] < n // 2, 0.0, 1.0).expand(B, n, h)
    constant, none = kind < 0.1, (kind >= 0.1) & (kind < 0.2)
    s = torch.where(constant, LEAST, s)
    m = torch.where(constant, torch.randn(B, n, h, generator=g, device="cuda") * torch.exp2(e), m)
    return torch.where(none[..., None], torch.zeros(2, dtype=BF, device="cuda"), _pairs(s, m)), constant | none


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("order", ["rising", "falling", "shuffled", "halves"])
@pytest.mark.parametrize("B,n,ql,hq,hkv,d,layout,page_size", [
    (120, 300, 1, 12, 1, 128, "NHD", 16), (200, 200, 1, 8, 2, 64, "HND", 5), (30, 400, 5, 8, 2, 128, "NHD", 16),
    (2, 700, 300, 16, 2, 128, "NHD", 24), (2, 450, 300, 16, 2, 64, "HND", 16),
])
def test_value_rows_of_unlike_scales(cuda, dtype, order, B, n, ql, hq, hkv, d, layout, page_size):
    g = _gen(7)
    codes = [_codes(g, (B, n, hkv, d)) for _ in range(2)]
    vp, flat = _mixed_pairs(g, order, B, n, hkv, 8)
    codes[1][flat] = 0
    kp = _plain_pairs(g, (B, n, hkv))
    q = torch.randn(B * ql, hq, d, generator=g, device="cuda")
    for causal in (True, False):
        _check(q, codes, kp, vp, ql, dtype, causal=causal, layout=layout, page_size=page_size)
    _check(3 * q, codes, kp, vp, ql, dtype, layout=layout, page_size=page_size)  # a sharp softmax


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ql,gain", [(1, 2.0 ** -12), (1, 2.0 ** -18), (5, 2.0 ** -20), (300, 2.0 ** -18)])
def test_small_fp16_queries_under_a_large_scale(cuda, d, ql, gain):
    """Queries down among fp16's least numbers keep all their bits in the logits."""
    B, n, h = 2 if ql > 8 else 60, 310, 2
    g = _gen(8)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    kp, vp = _plain_pairs(g, (B, n, h)), _plain_pairs(g, (B, n, h))
    q = torch.randn(B * ql, 16, d, generator=g, device="cuda") * gain
    _check(q, codes, kp, vp, ql, FP, scale=d ** -0.5 / gain)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ql", [1, 5, 300])
@pytest.mark.parametrize("keys,queries,scale", [
    (2.0 ** 110, 2.0 ** -110, 1.0), (2.0 ** 122, 2.0 ** -122, 1.0), (2.0 ** 124, 2.0 ** -100, 2.0 ** -24),
    (2.0 ** 124, 2.0 ** -100, -(2.0 ** -24)),
    (2.0 ** -100, 2.0 ** 110, 2.0 ** -10), (2.0 ** -118, 2.0 ** 117, 1.0), (1.0, 2.0 ** -60, 2.0 ** 60), (1.0, 2.0 ** 60, 2.0 ** -60),
])
def test_key_rows_and_queries_at_the_ends_of_their_range(cuda, d, ql, keys, queries, scale):
    B, n, h = 2 if ql > 8 else 60, 310, 2
    g = _gen(9)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    kp, vp = _plain_pairs(g, (B, n, h), keys), _plain_pairs(g, (B, n, h))
    q = torch.randn(B * ql, 16, d, generator=g, device="cuda") * queries
    _check(q, codes, kp, vp, ql, BF, scale=scale * d ** -0.5)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("ql", [1, 5, 300])
def test_a_scale_of_zero_weighs_all_keys_alike(cuda, dtype, ql):
    B, n, h, d = 2 if ql > 8 else 60, 310, 2, 128
    g = _gen(10)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    kp, vp = _plain_pairs(g, (B, n, h)), _plain_pairs(g, (B, n, h))
    _check(torch.randn(B * ql, 16, d, generator=g, device="cuda"), codes, kp, vp, ql, dtype, scale=0.0)


@pytest.mark.parametrize("value", [-1e20, 1e26, 1e-30])
@pytest.mark.parametrize("ql", [1, 8, 1200])
def test_constant_values_of_any_size(cuda, value, ql):
    """The same cache through both kernels: the value, off by its rounding and the sums'."""
    B, n, h, d = 1, 2000, 2, 128
    g = _gen(11)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    codes[1].zero_()
    vp = torch.tensor([LEAST, value], device="cuda").to(BF).expand(B, n, h, 2)
    _check(torch.randn(ql, 16, d, generator=g, device="cuda"), codes, _plain_pairs(g, (B, n, h)), vp, ql, BF)


@pytest.mark.parametrize("order", ["all", "mixed"])
@pytest.mark.parametrize("scale", [2.0 ** -75, 2.0 ** -92, 2.0 ** 90])
@pytest.mark.parametrize("ql", [1, 300])
def test_values_of_very_small_and_very_large_scales(cuda, order, scale, ql):
    B, n, h, d = 2 if ql > 8 else 60, 450, 2, 128
    g = _gen(12)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    vp = _plain_pairs(g, (B, n, h), scale)
    if order == "mixed":  # constant rows of the same size between them
        flat = torch.rand(B, n, h, generator=g, device="cuda") < 0.5
        vp = torch.where(flat[..., None], torch.tensor([LEAST, 3 * scale], device="cuda").to(BF), vp)
        codes[1][flat] = 0
    _check(torch.randn(B * ql, 16, d, generator=g, device="cuda"), codes, _plain_pairs(g, (B, n, h)), vp, ql, BF)


@pytest.mark.parametrize("dtype,scale", [(FP, 100.0), (BF, 100.0), (BF, 2.0 ** 40), (BF, 2.0 ** 85)])
@pytest.mark.parametrize("first", ["zero pairs", "zeros", "wide"])
@pytest.mark.parametrize("ql", [1, 300])
def test_wide_values_beside_a_long_stretch_of_nothing(cuda, dtype, scale, first, ql):
    """Half a context of rows that hold zeros, half of wide ones, cut into parts: the zeros keep their share of the weight."""
    B, n, h, d = 2, 2500, 2, 128
    g = _gen(13)
    codes = [_codes(g, (B, n, h, d)) for _ in range(2)]
    vp = _plain_pairs(g, (B, n, h), scale)
    none = torch.arange(n, device="cuda") < n // 2
    none = (~none if first == "wide" else none)[None, :, None].expand(B, n, h)
    vp = torch.where(none[..., None], torch.tensor([0.0 if first == "zero pairs" else LEAST, 0.0], device="cuda").to(BF), vp)
    codes[1][none] = 0
    q = torch.randn(B * ql, 16, d, generator=g, device="cuda")
    for causal in (True, False):
        _check(q, codes, _plain_pairs(g, (B, n, h)), vp, ql, dtype, causal=causal)
