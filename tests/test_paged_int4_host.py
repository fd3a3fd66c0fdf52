"""The 4-bit cache's operators without a GPU: argument checks, fake kernels, the C entry points' refusals, and the
test reference's own arithmetic."""
from __future__ import annotations

import ctypes
import math
import re
from fractions import Fraction
from pathlib import Path

import pytest
import torch

import kv_int4_ref as ref
import mas_b200
from mas_b200 import _lib

M = "meta"
BF = torch.bfloat16
I32 = torch.int32
HEADER = Path(__file__).resolve().parents[1] / "include" / "mas_b200.h"


def _cache(pages=4, ps=16, heads=2, d=128, layout="NHD", device=M):
    return mas_b200.empty_paged_kv_cache_int4(pages, ps, heads, d, layout, device=device)


def _append(**kw):
    a = dict(append_key=torch.empty(3, 2, 128, dtype=BF, device=M), append_value=torch.empty(3, 2, 128, dtype=BF, device=M),
             batch_indices=torch.empty(3, dtype=I32, device=M), positions=torch.empty(3, dtype=I32, device=M),
             paged_kv_cache=_cache(), kv_indices=torch.empty(4, dtype=I32, device=M), kv_indptr=torch.empty(3, dtype=I32, device=M),
             kv_last_page_len=torch.empty(2, dtype=I32, device=M))
    a.update(kw)
    return mas_b200.append_paged_kv_cache_int4(**a)


def _read(**kw):
    a = dict(batch_indices=torch.empty(3, dtype=I32, device=M), positions=torch.empty(3, dtype=I32, device=M),
             paged_kv_cache=_cache(), kv_indices=torch.empty(4, dtype=I32, device=M), kv_indptr=torch.empty(3, dtype=I32, device=M))
    a.update(kw)
    return mas_b200.read_paged_kv_cache_int4(**a)


def _attend(**kw):
    a = dict(query=torch.empty(3, 4, 128, dtype=BF, device=M), paged_kv_cache=_cache(),
             block_tables=torch.empty(2, 5, dtype=I32, device=M), seq_lens=torch.empty(2, dtype=I32, device=M),
             cum_seq_lens_q=torch.empty(3, dtype=I32, device=M))
    a.update(kw)
    return mas_b200.paged_attention_int4(**a)


def _allocate(**kw):
    a = dict(append_lens=torch.empty(2, dtype=I32, device=M), seq_lens=torch.empty(2, dtype=I32, device=M),
             block_tables=torch.empty(2, 5, dtype=I32, device=M), free_pages=torch.empty(9, dtype=I32, device=M),
             num_free=torch.empty(1, dtype=I32, device=M), page_size=16, max_tokens=7)
    a.update(kw)
    return mas_b200.allocate_paged_kv(**a)


def _release(**kw):
    a = dict(keep_lens=torch.empty(2, dtype=I32, device=M), seq_lens=torch.empty(2, dtype=I32, device=M),
             block_tables=torch.empty(2, 5, dtype=I32, device=M), free_pages=torch.empty(9, dtype=I32, device=M),
             num_free=torch.empty(1, dtype=I32, device=M), page_size=16)
    a.update(kw)
    return mas_b200.release_paged_kv(**a)


def test_shapes_of_the_results():
    k, v, pairs = _cache(pages=3, ps=5, heads=7, d=64, layout="HND")
    assert k.shape == v.shape == (3, 7, 5, 32) and pairs.shape == (3, 7, 5, 4)
    assert k.dtype == torch.uint8 and pairs.dtype == BF
    assert _append() is None and _release() is None
    key, value = _read(dtype=torch.float16)
    assert key.shape == value.shape == (3, 2, 128) and key.dtype == torch.float16
    assert _attend().shape == (3, 4, 128)
    out, lse = _attend(query=torch.empty(3, 4 * 128, dtype=BF, device=M), return_lse=True)
    assert out.shape == (3, 512) and lse.shape == (3, 4) and lse.dtype == torch.float32
    maps = _allocate()
    assert [tuple(t.shape) for t in maps] == [(3,), (7,), (7,), (2,)]
    assert _allocate(out=maps).positions is maps.positions


def t(*shape, dtype=I32, device=M):
    return torch.empty(shape, dtype=dtype, device=device)


REFUSALS = [
    (_append, dict(kv_layout="NDH"), KeyError),
    (_append, dict(paged_kv_cache=_cache()[:2]), KeyError),
    (_append, dict(append_value=t(3, 2, 64, dtype=BF)), ValueError),
    (_append, dict(append_value=t(3, 2, 128, dtype=torch.float16)), ValueError),
    (_append, dict(append_key=t(3, 2, 128, dtype=torch.float32), append_value=t(3, 2, 128, dtype=torch.float32)), ValueError),
    (_append, dict(append_key=t(3, 4, 128, dtype=BF), append_value=t(3, 4, 128, dtype=BF)), ValueError),
    (_append, dict(append_key=t(3, 2, 256, dtype=BF)[..., ::2]), ValueError),
    (_append, dict(batch_indices=t(4)), ValueError),
    (_append, dict(kv_last_page_len=t(3)), ValueError),
    (_append, dict(paged_kv_cache=(t(4, 16, 2, 48, dtype=torch.uint8),) * 2 + (t(4, 2, 16, 4, dtype=BF),)), ValueError),
    (_append, dict(paged_kv_cache=(t(4, 16, 2, 64, dtype=torch.int8),) * 2 + (t(4, 2, 16, 4, dtype=BF),)), ValueError),
    (_append, dict(paged_kv_cache=(t(4, 16, 2, 64, dtype=torch.uint8),) * 2 + (t(4, 16, 2, 4, dtype=BF),)), ValueError),
    (_append, dict(paged_kv_cache=(t(4, 16, 2, 64, dtype=torch.uint8),) * 2 + (t(4, 2, 16, 8, dtype=BF)[..., ::2],)), ValueError),
    (_append, dict(paged_kv_cache=(t(4, 16, 2, 72, dtype=torch.uint8)[..., :64],) * 2 + (t(4, 2, 16, 4, dtype=BF),)), ValueError),
    (_append, dict(append_key=t(3, 2, 128, dtype=BF, device="cpu"), append_value=t(3, 2, 128, dtype=BF, device="cpu")), RuntimeError),
    (_read, dict(dtype=torch.float32), ValueError),
    (_read, dict(positions=t(2)), ValueError),
    (_read, dict(out=(t(3, 2, 128, dtype=BF), t(3, 2, 128, dtype=torch.float16))), ValueError),
    (_read, dict(out=(t(3, 2, 64, dtype=BF), t(3, 2, 64, dtype=BF))), ValueError),
    (_read, dict(kv_indptr=t(3, device="cpu")), RuntimeError),
    (_attend, dict(query=t(3, 5, 128, dtype=BF)), ValueError),
    (_attend, dict(query=t(3, 4, 64, dtype=BF)), ValueError),
    (_attend, dict(query=t(3, 4, 128, dtype=torch.float32)), ValueError),
    (_attend, dict(query=t(3, 500, dtype=BF)), ValueError),
    (_attend, dict(cum_seq_lens_q=None), ValueError),
    (_attend, dict(cum_seq_lens_q=t(2)), ValueError),
    (_attend, dict(seq_lens=t(2, dtype=torch.int64)), ValueError),
    (_attend, dict(block_tables=t(3, 5)), ValueError),
    (_attend, dict(block_tables=t(5, 2).t()), ValueError),
    (_attend, dict(out=t(3, 4, 128, dtype=torch.float16)), ValueError),
    (_attend, dict(kv_layout="HND"), ValueError),
    (_attend, dict(block_tables=t(2, 5, device="cpu"), seq_lens=t(2)), RuntimeError),
    (_allocate, dict(append_lens=t(3)), ValueError),
    (_allocate, dict(append_lens=t(2, dtype=torch.float32)), ValueError),
    (_allocate, dict(seq_lens=t(2, dtype=torch.int64)), ValueError),
    (_allocate, dict(num_free=t(2)), ValueError),
    (_allocate, dict(page_size=0), ValueError),
    (_allocate, dict(max_tokens=-1), ValueError),
    (_allocate, dict(free_pages=t(9, 2)[:, 0]), ValueError),
    (_allocate, dict(block_tables=t(1, 5).expand(2, 5)), ValueError),
    (_allocate, dict(append_lens=t(8193), seq_lens=t(8193), block_tables=t(8193, 1)), ValueError),
    (_allocate, dict(out=(t(3), t(7), t(6), t(2))), ValueError),
    (_allocate, dict(free_pages=t(9, device="cpu")), RuntimeError),
    (_release, dict(keep_lens=t(1)), ValueError),
    (_release, dict(block_tables=t(2, 5, dtype=torch.int64)), ValueError),
    (_release, dict(num_free=t(1, device="cpu")), RuntimeError),
]


@pytest.mark.parametrize("fn,kw,exc", REFUSALS)
def test_refusals(fn, kw, exc):
    with pytest.raises(exc):
        fn(**kw)


def _onto(x, device):
    """Meta tensors as tensors of that layout on `device`; others as they are."""
    if torch.is_tensor(x):
        return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=device) if x.device.type == "meta" else x
    return tuple(_onto(y, device) for y in x) if isinstance(x, tuple) else x


@pytest.mark.gpu
@pytest.mark.parametrize("fn,kw,exc", REFUSALS)
def test_refusals_of_cuda_calls(cuda, monkeypatch, fn, kw, exc):
    """The operators' own checks of CUDA tensors raise what the Python checks raise; nothing is launched."""
    import mas_b200.paged_int4 as module

    for name in ("append_paged_kv_cache_int4", "read_paged_kv_cache_int4", "paged_attention_int4", "allocate_paged_kv",
                 "release_paged_kv"):
        real = getattr(module, name)
        monkeypatch.setattr(mas_b200, name, lambda real=real, **a: real(**{k: _onto(v, cuda) for k, v in a.items()}))
    with pytest.raises(exc):
        fn(**kw)
    torch.cuda.synchronize()


def test_no_cpu_implementation():
    cache = _cache(device="cpu")
    with pytest.raises(NotImplementedError):
        _attend(query=t(3, 4, 128, dtype=BF, device="cpu"), paged_kv_cache=cache, block_tables=t(2, 5, device="cpu"),
                seq_lens=t(2, device="cpu"), cum_seq_lens_q=t(3, device="cpu"))


def test_struct_layout_and_status_bit_match_header():
    text = HEADER.read_text()
    body = re.search(r"typedef struct MasInt4KVCache \{(.*?)\} MasInt4KVCache;", text, re.S).group(1)
    assert re.findall(r"(\w+);", body) == [f for f, _ in _lib.Int4KVCache._fields_]
    assert ctypes.sizeof(_lib.Int4KVCache) == 72
    assert int(re.search(r"MAS_STATUS_KV_ALLOC_REFUSED (\d+)", text).group(1)) == _lib.STATUS_KV_ALLOC_REFUSED


L, P = _lib.lib, 0x1000  # a non-null pointer value: the checks come before any use of it


def _kv(**kw):
    a = dict(k_codes=P, v_codes=P, pairs=P, num_pages=4, page_size=16, stride_page=2048, stride_entry=128, stride_head=64,
             pair_stride_page=128)
    a.update(kw)
    return ctypes.byref(_lib.Int4KVCache(**a))


def _c_append(kv=None, d=128, T=3, heads=2, dtype=0, pdt=4, key=P, read=False, num_indices=4):
    f = L.mas_read_paged_kv_cache_int4 if read else L.mas_append_paged_kv_cache_int4
    return f(key, P, P, P, pdt, _kv() if kv is None else kv, P, num_indices, P, 2, T, heads, d, 256, 128, 256, 128, dtype, None, 0, None)


def _c_attend(kv=None, q=P, B=2, T=2, hq=4, hkv=2, d=128, table=5, blocks=5, cum=None, dtype=0, work=P, seq=P, qs=512, tab=P):
    return L.mas_paged_attention_int4(q, P, None, _kv() if kv is None else kv, tab, table, blocks, seq, cum, B, T, hq, hkv, d, qs, 128,
                                      512, 128, 0.1, 1, dtype, work, 1 << 40, None, 0, None)


def _c_alloc(B=2, blocks=5, stride=5, ps=16, tokens=4, cap=9, num=P, lens=P):
    return L.mas_allocate_paged_kv(lens, P, P, P, num, P, P, P, P, B, blocks, stride, ps, tokens, cap, None, 0, None)


def _c_release(B=2, blocks=5, stride=5, ps=16, cap=9):
    return L.mas_release_paged_kv(P, P, P, P, P, B, blocks, stride, ps, cap, None, 0, None)


@pytest.mark.parametrize("call,code", [
    (lambda: _c_append(dtype=2), -2), (lambda: _c_append(pdt=1), -2), (lambda: _c_append(d=96), -3), (lambda: _c_append(T=-1), -1),
    (lambda: _c_append(heads=0), -1), (lambda: _c_append(key=None), -1), (lambda: _c_append(num_indices=-1), -1),
    (lambda: _c_append(kv=_kv(k_codes=None)), -1), (lambda: _c_append(kv=_kv(page_size=0)), -1),
    (lambda: _c_append(kv=_kv(stride_head=72)), -1), (lambda: _c_append(kv=_kv(v_codes=P + 8)), -1),
    (lambda: _c_append(kv=_kv(pairs=P + 4)), -1), (lambda: _c_append(kv=_kv(pair_stride_page=127)), -1),
    (lambda: _c_append(read=True, d=32), -3), (lambda: _c_append(read=True, key=None), -1),
    (lambda: _c_attend(hq=5), -1), (lambda: _c_attend(d=256), -3), (lambda: _c_attend(dtype=3), -2), (lambda: _c_attend(T=3), -1),
    (lambda: _c_attend(B=-1), -1), (lambda: _c_attend(table=4), -1), (lambda: _c_attend(q=None), -1), (lambda: _c_attend(seq=None), -1),
    (lambda: _c_attend(T=1 << 30, cum=P), -3), (lambda: _c_attend(tab=None), -1), (lambda: _c_attend(qs=-1), -1),
    (lambda: _c_alloc(B=-1), -1), (lambda: _c_alloc(B=8193), -3), (lambda: _c_alloc(stride=4), -1), (lambda: _c_alloc(ps=0), -1),
    (lambda: _c_alloc(tokens=-1), -1), (lambda: _c_alloc(cap=-1), -1), (lambda: _c_alloc(num=None), -1), (lambda: _c_alloc(lens=None), -1),
    (lambda: _c_release(B=8193), -3), (lambda: _c_release(blocks=-1), -1),
    (lambda: L.mas_paged_attention_int4_workspace(128, None), -1),
    (lambda: L.mas_paged_attention_int4_workspace(96, ctypes.byref(ctypes.c_int64())), -3),
])
def test_c_entry_points_reject_before_launch(call, code):
    assert call() == code


def test_c_entry_points_with_nothing_to_do():
    assert _c_append(T=0) == 0 and _c_append(T=0, read=True) == 0
    assert _c_attend(B=0, T=0) == 0 and _c_attend(T=0, cum=P) == 0
    assert _c_release(B=0) == 0


# The reference the GPU tests compare with, on rows whose form is known.
def test_reference_quantiser():
    codes, s, m = ref.quantise_row(torch.tensor([0.0, 15.0, 7.5, 0.5, 0.499]))
    assert (s, m) == (1.0, 0.0) and codes == [0, 15, 8, 1, 0]
    codes, s, m = ref.quantise_row(torch.full((4,), -3.0))
    assert (s, m) == (2.0 ** -126, -3.0) and codes == [0] * 4
    codes, s, m = ref.quantise_row(torch.tensor([1.0, 1.0009765625], dtype=torch.float16))
    assert m == 1.0 and 15 * s >= 0.0009765625 and codes == [0, 15]
    assert math.isnan(ref.quantise_row(torch.tensor([1.0, math.inf]))[1])
    big = 3.3895313892515355e38
    codes, s, m = ref.quantise_row(torch.tensor([-big, 0.0, big]))
    assert codes == [0, 8, 15] or codes == [0, 7, 15]
    assert Fraction(m) + 15 * Fraction(s) >= Fraction(big) and s < 2 * big / 15 * (1 + 2 ** -7)


def test_reference_pages_round_trip():
    lens, new = [0, 5, 16, 31], [3, 0, 1, 20]
    table, free = [[-1] * 5 for _ in lens], list(range(40, 60))
    ok, cum, bi, pos, last, now, tab, num = ref.allocate(new, lens, table, free, 20, 16, 30)
    assert ok and cum == [0, 3, 3, 4, 24] and bi[:5] == [0, 0, 0, 2, 3] and bi[24:] == [-1] * 6 and last == [3, 5, 1, 3]
    assert tab[0][0] == 59 and tab[2][1] == 58 and tab[3][2:4] == [57, 56] and num == 16
    ok, back, fl, n = ref.release(lens, now, tab, free, num, 16)
    assert ok and back == lens and fl == free and n == 20
