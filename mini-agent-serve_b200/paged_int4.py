"""The paged KV cache in 4 bits: page allocation on the GPU, the quantising append with its read-back, and
the attention that reads the cache.

A step of a decoder whose cache is held in 4 bits, beside the ops of ops.py::

    cache = empty_paged_kv_cache_int4(num_pages, page_size, num_kv_heads, head_dim)   # once, a layer
    maps = allocate_paged_kv(append_lens, seq_lens, block_tables, free_pages, num_free, page_size, max_tokens)
    ... per layer ...
    apply_rope_with_cos_sin_cache_inplace(maps.positions, q, k, head_dim, cos_sin_cache)
    append_paged_kv_cache_int4(k_heads, v_heads, maps.batch_indices, maps.positions, cache, block_tables.flatten(),
                               kv_indptr, maps.kv_last_page_len)            # kv_indptr = arange(B + 1) * max_blocks
    out = paged_attention_int4(q_heads, cache, block_tables, seq_lens, maps.cum_append_lens)
    ... drafts rejected, requests finished ...
    release_paged_kv(keep_lens, seq_lens, block_tables, free_pages, num_free, page_size)

The metadata are the tensors the engine already passes around (miniagentserve/models/devstral2/devstral2.py:118-136,
:283-290), and the append takes the arguments of append_paged_kv_cache with the 4-bit cache in its place.
Attention stands where Devstral2Attention.forward calls flashinfer's paged attention (devstral2.py:184-213).

The cache of a layer is the tuple (k_codes, v_codes, pairs). A row is one token's k or v of one kv head: head_dim
codes c of 4 bits, two a byte (element 2i in the low half), and a bf16 pair (scale s, minimum m); its values are
c * s + m. The codes are uint8 [pages, page_size, heads, head_dim / 2] (NHD) or [pages, heads, page_size,
head_dim / 2] (HND); the pairs bf16 [pages, heads, page_size, 4], (k s, k m, v s, v m), under either layout.
At head_dim 128 that is 136 bytes a token and kv head, against 512 in 16 bits.

As in ops.py, each function stands over a `mas_b200::*` operator that launches on the current stream, is opaque to
torch.compile and can be captured into a CUDA graph; there is no CPU implementation. CUDA calls are checked by the operator
itself (csrc/torch_ops.cpp), with the exceptions the checks here raise for tensors of other devices: a decode step is a few
microseconds of kernels, and these checks took ten to twenty in Python.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib  # noqa: F401  (loads the operators)
from .ops import _ID_DTYPES, _act_code, _check_device, _heads

__all__ = [
    "PagedKVMaps",
    "allocate_paged_kv",
    "release_paged_kv",
    "empty_paged_kv_cache_int4",
    "append_paged_kv_cache_int4",
    "read_paged_kv_cache_int4",
    "paged_attention_int4",
]

MAX_REQUESTS = 8192  # a page allocation scans all lengths in one thread block's shared memory
HEAD_DIMS = (64, 128)

_OP_ALLOCATE = torch.ops.mas_b200.allocate_paged_kv.default
_OP_ALLOCATE_OUT = torch.ops.mas_b200.allocate_paged_kv_out.default
_OP_RELEASE = torch.ops.mas_b200.release_paged_kv.default
_OP_APPEND = torch.ops.mas_b200.append_paged_kv_cache_int4.default
_OP_READ = torch.ops.mas_b200.read_paged_kv_cache_int4.default
_OP_READ_OUT = torch.ops.mas_b200.read_paged_kv_cache_int4_out.default
_OP_ATTENTION = torch.ops.mas_b200.paged_attention_int4.default
_OP_ATTENTION_OUT = torch.ops.mas_b200.paged_attention_int4_out.default


@torch.library.register_fake("mas_b200::allocate_paged_kv")
def _(append_lens, seq_lens, block_tables, free_pages, num_free, page_size, max_tokens, enable_pdl):
    def new(n):
        return seq_lens.new_empty((n,), dtype=torch.int32)
    return new(seq_lens.shape[0] + 1), new(max_tokens), new(max_tokens), new(seq_lens.shape[0])


@torch.library.register_fake("mas_b200::allocate_paged_kv_out")
def _(append_lens, seq_lens, block_tables, free_pages, num_free, cum_append_lens, batch_indices, positions,
      kv_last_page_len, page_size, max_tokens, enable_pdl) -> None:
    return None


@torch.library.register_fake("mas_b200::release_paged_kv")
def _(keep_lens, seq_lens, block_tables, free_pages, num_free, page_size, enable_pdl) -> None:
    return None


@torch.library.register_fake("mas_b200::append_paged_kv_cache_int4")
def _(k, v, batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd, enable_pdl) -> None:
    return None


@torch.library.register_fake("mas_b200::read_paged_kv_cache_int4")
def _(batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, dtype, hnd, enable_pdl):
    shape = (batch_indices.shape[0], k_codes.shape[1 if hnd else 2], 2 * k_codes.shape[3])
    return k_codes.new_empty(shape, dtype=dtype), k_codes.new_empty(shape, dtype=dtype)


@torch.library.register_fake("mas_b200::read_paged_kv_cache_int4_out")
def _(k, v, batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd, enable_pdl) -> None:
    return None


@torch.library.register_fake("mas_b200::paged_attention_int4")
def _(query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, sm_scale, causal, hnd, return_lse, enable_pdl):
    heads = query.shape[1] if query.dim() == 3 else query.shape[1] // (2 * k_codes.shape[3])
    return (torch.empty(query.shape, dtype=query.dtype, device=query.device),
            query.new_empty((query.shape[0] if return_lse else 0, heads), dtype=torch.float32))


@torch.library.register_fake("mas_b200::paged_attention_int4_out")
def _(out, lse, query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, sm_scale, causal, hnd,
      enable_pdl) -> None:
    return None


def _check_int32(name: str, t: torch.Tensor, shape: Optional[tuple] = None) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")


def _check_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor) -> int:
    _check_int32("seq_lens", seq_lens)
    if seq_lens.dim() != 1:
        raise ValueError("seq_lens must be (batch_size,)")
    if (block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.shape[0] != seq_lens.shape[0]
            or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1)):
        raise ValueError("block_tables must be an int32 (batch_size, max_blocks) tensor, contiguous within a row")
    if block_tables.shape[0] > 1 and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError("block_tables' rows must not overlap")
    return seq_lens.shape[0]


# ------------------------------------------------------------------------------------------------
# Pages.
# ------------------------------------------------------------------------------------------------
class PagedKVMaps(NamedTuple):
    """What a step's kernels need to place its new tokens (all int32)."""

    cum_append_lens: torch.Tensor   # (batch_size + 1,) exclusive sum of append_lens: the queries' cum_seq_lens_q
    batch_indices: torch.Tensor     # (max_tokens,) each new token's request, -1 behind the last token
    positions: torch.Tensor         # (max_tokens,) its position in the request, 0 behind the last token
    kv_last_page_len: torch.Tensor  # (batch_size,) tokens on the request's last page after the step


def _check_pages(seq_lens, block_tables, free_pages, num_free, page_size) -> int:
    batch = _check_tables(block_tables, seq_lens)
    _check_int32("free_pages", free_pages)
    _check_int32("num_free", num_free, (1,))
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be (capacity,)")
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    if batch > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests a call, got {batch}")
    return batch


def allocate_paged_kv(append_lens: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
                      free_pages: torch.Tensor, num_free: torch.Tensor, page_size: int, max_tokens: int,
                      out: Optional[PagedKVMaps] = None, enable_pdl: Optional[bool] = None) -> PagedKVMaps:
    r"""Takes the pages a step's new tokens need and maps the tokens, without the host knowing a length.

    ``append_lens[b]`` tokens join the ``seq_lens[b]`` of request ``b``. Pages come off the stack `free_pages`, of
    which the first ``num_free[0]`` entries are free, last first, to the requests in order; they are written behind
    the used entries of ``block_tables[b]``. `seq_lens`, `block_tables` and `num_free` (all int32) are updated in
    place, so a captured step carries its state along. Returns the token maps, sized for `max_tokens` (entries
    behind the step's last token name no request: -1), in new tensors or in `out`'s.

    A step that does not fit (free pages, table columns, `max_tokens`, a negative length) takes nothing: the state
    stays as it is, the maps say that no token has a place, and STATUS_KV_ALLOC_REFUSED is set in the device
    status word (`read_status`). At most 8192 requests.
    """
    pdl = True if enable_pdl is None else bool(enable_pdl)
    if not seq_lens.is_cuda:
        _check_allocate(append_lens, seq_lens, block_tables, free_pages, num_free, page_size, max_tokens, out)
    if out is None:
        return PagedKVMaps(*_OP_ALLOCATE(append_lens, seq_lens, block_tables, free_pages, num_free, page_size, max_tokens, pdl))
    _OP_ALLOCATE_OUT(append_lens, seq_lens, block_tables, free_pages, num_free, *out, page_size, max_tokens, pdl)
    return PagedKVMaps(*out)


def _check_allocate(append_lens, seq_lens, block_tables, free_pages, num_free, page_size, max_tokens, out) -> None:
    batch = _check_pages(seq_lens, block_tables, free_pages, num_free, page_size)
    if append_lens.shape != (batch,) or append_lens.dtype not in _ID_DTYPES:
        raise ValueError("append_lens must be an int32 or int64 (batch_size,) tensor")
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    maps = {} if out is None else PagedKVMaps(*out)._asdict()
    for (name, t), n in zip(maps.items(), (batch + 1, max_tokens, max_tokens, batch)):
        _check_int32(name, t, (n,))
    _check_device(seq_lens, append_lens=append_lens, block_tables=block_tables, free_pages=free_pages,
                  num_free=num_free, **maps)


def release_paged_kv(keep_lens: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor,
                     free_pages: torch.Tensor, num_free: torch.Tensor, page_size: int,
                     enable_pdl: Optional[bool] = None) -> None:
    r"""Cuts each request to ``keep_lens[b] <= seq_lens[b]`` tokens (0: it has finished) and gives its pages back.

    The inverse of `allocate_paged_kv`: `seq_lens`, `num_free` and the stack `free_pages` are updated in place, and
    releasing what the last call took leaves the stack as it was. `block_tables` stays as it is. Pages that several
    requests share must not be released through each of them. A call that does not fit changes nothing and sets
    STATUS_KV_ALLOC_REFUSED.
    """
    if not seq_lens.is_cuda:
        batch = _check_pages(seq_lens, block_tables, free_pages, num_free, page_size)
        if keep_lens.shape != (batch,) or keep_lens.dtype not in _ID_DTYPES:
            raise ValueError("keep_lens must be an int32 or int64 (batch_size,) tensor")
        _check_device(seq_lens, keep_lens=keep_lens, block_tables=block_tables, free_pages=free_pages, num_free=num_free)
    _OP_RELEASE(keep_lens, seq_lens, block_tables, free_pages, num_free, page_size,
                True if enable_pdl is None else bool(enable_pdl))


# ------------------------------------------------------------------------------------------------
# The cache.
# ------------------------------------------------------------------------------------------------
def empty_paged_kv_cache_int4(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                              kv_layout: str = "NHD", device="cuda") -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One layer's cache, (k_codes, v_codes, pairs), all zeros: every row reads as zeros."""
    hnd = _is_hnd(kv_layout)
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    inner = (page_size, num_kv_heads) if not hnd else (num_kv_heads, page_size)
    codes = [torch.zeros((num_pages, *inner, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
    return codes[0], codes[1], torch.zeros((num_pages, num_kv_heads, page_size, 4), dtype=torch.bfloat16, device=device)


def _is_hnd(kv_layout: str) -> bool:
    if kv_layout not in ("NHD", "HND"):
        raise KeyError(f"Invalid kv_layout {kv_layout}")
    return kv_layout == "HND"


def _parts(paged_kv_cache):
    if not isinstance(paged_kv_cache, (tuple, list)) or len(paged_kv_cache) != 3:
        raise KeyError("paged_kv_cache must be (k_codes, v_codes, pairs)")
    return paged_kv_cache


def _check_cache(k_codes, v_codes, pairs, hnd: bool):
    """(heads, head_dim) of a cache whose layout the kernels take."""
    if k_codes.dim() != 4 or k_codes.shape != v_codes.shape:
        raise ValueError("k/v codes must be 4-D with identical shapes")
    if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8 or pairs.dtype != torch.bfloat16:
        raise ValueError("k/v codes must be uint8 and pairs bfloat16")
    pages, page_size, heads = k_codes.shape[0], k_codes.shape[1], k_codes.shape[2]
    if hnd:
        page_size, heads = heads, page_size
    head_dim = 2 * k_codes.shape[3]
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if page_size < 1 or heads < 1:
        raise ValueError("page_size and the number of heads must be positive")
    if tuple(pairs.shape) != (pages, heads, page_size, 4):
        raise ValueError(f"pairs must have shape {(pages, heads, page_size, 4)}, got {tuple(pairs.shape)}")
    for n in range(1, 4):
        if pairs.shape[n] > 1 and pairs.stride(n) != (page_size * 4, 4, 1)[n - 1]:
            raise ValueError("pairs must be contiguous within a page")
    if pages > 1 and (pairs.stride(0) % 4 or pairs.stride(0) < heads * page_size * 4):
        raise ValueError("pairs' pages must not overlap and lie a multiple of 4 elements apart")
    for n in range(4):
        if k_codes.shape[n] > 1:
            if k_codes.stride(n) != v_codes.stride(n):
                raise ValueError("k/v codes must have identical strides")
            if k_codes.stride(n) % 16 if n < 3 else k_codes.stride(n) != 1:
                raise ValueError("k/v codes must be contiguous in the last dimension, the others' strides multiples of 16")
    _check_device(k_codes, v_codes=v_codes, pairs=pairs)
    return heads, head_dim


def _check_rows(batch_indices, positions, kv_indptr, tokens: int) -> None:
    if batch_indices.shape != (tokens,) or positions.shape != (tokens,):
        raise ValueError("batch_indices and positions must have one entry per token")
    if kv_indptr.dim() != 1 or kv_indptr.shape[0] < 1:
        raise ValueError("kv_indptr must have batch_size + 1 entries")
    if positions.dtype not in _ID_DTYPES:
        raise ValueError("positions must be int32 or int64")


def append_paged_kv_cache_int4(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                               positions: torch.Tensor, paged_kv_cache, kv_indices: torch.Tensor,
                               kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor, kv_layout: str = "NHD",
                               enable_pdl: Optional[bool] = None) -> None:
    r"""Quantises each token's k and v rows to 4 bits and stores them in the paged cache.

    `append_paged_kv_cache` with the cache ``(k_codes, v_codes, pairs)``: the same arguments, the same slot
    (entry ``p % page_size`` of page ``kv_indices[kv_indptr[b] + p // page_size]``), the same handling of an index
    out of range. A row x gets the minimum ``m``, the largest bf16 not above ``min(x)``, the scale ``s``, the least bf16
    with ``m + 15 s >= max(x)`` (and at least 2^-126), and the codes ``floor((x - m) / s + 1/2)``, the difference taken in
    fp32; a row that holds a NaN or an infinity reads as NaN. A token with ``batch_indices[i] == -1`` (the padding that
    `allocate_paged_kv` leaves) is skipped. Two tokens must not name one slot. head_dim is 64 or 128.
    """
    hnd = _is_hnd(kv_layout)
    k_codes, v_codes, pairs = _parts(paged_kv_cache)
    if kv_last_page_len.dim() != 1 or kv_indptr.dim() != 1 or kv_indptr.shape[0] != kv_last_page_len.shape[0] + 1:
        raise ValueError("kv_indptr must have batch_size + 1 entries, kv_last_page_len batch_size")
    if not append_key.is_cuda:
        heads, head_dim = _check_cache(k_codes, v_codes, pairs, hnd)
        if append_key.dim() != 3 or append_value.shape != append_key.shape:
            raise ValueError("append_key and append_value must be (nnz, num_kv_heads, head_dim) and equal in shape")
        if append_key.dtype != append_value.dtype:
            raise ValueError("append_key and append_value must share one dtype")
        _act_code(append_key)
        if tuple(append_key.shape[1:]) != (heads, head_dim):
            raise ValueError(f"cache heads/head_dim {(heads, head_dim)} differ from {tuple(append_key.shape[1:])}")
        if append_key.stride(2) != 1 or append_value.stride(2) != 1:
            raise ValueError("append_key and append_value must be contiguous in head_dim")
        _check_rows(batch_indices, positions, kv_indptr, append_key.shape[0])
        _check_device(append_key, append_value=append_value, batch_indices=batch_indices, positions=positions,
                      k_codes=k_codes, kv_indices=kv_indices, kv_indptr=kv_indptr)
    _OP_APPEND(append_key, append_value, batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd,
               True if enable_pdl is None else bool(enable_pdl))


def read_paged_kv_cache_int4(batch_indices: torch.Tensor, positions: torch.Tensor, paged_kv_cache,
                             kv_indices: torch.Tensor, kv_indptr: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                             kv_layout: str = "NHD", out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                             enable_pdl: Optional[bool] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    r"""The k and v rows the cache holds for the named tokens, ``(nnz, num_kv_heads, head_dim)`` each.

    The inverse of `append_paged_kv_cache_int4`: ``c * s + m`` in fp32, rounded once to `dtype` (bfloat16 or float16;
    a value past its largest finite one reads as that one). For what must have a cached prefix in 16 bits: a prompt
    kernel of another library, a check, a copy to a 16-bit cache. A padding row (-1) or one out of range (flagged as
    in the append) reads as zeros. `out` takes two tensors that share shape and dtype (any strides, contiguous in head_dim).
    """
    hnd = _is_hnd(kv_layout)
    k_codes, v_codes, pairs = _parts(paged_kv_cache)
    pdl = True if enable_pdl is None else bool(enable_pdl)
    if out is None and dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported dtype {dtype}; expected bfloat16 or float16")
    if not k_codes.is_cuda:
        _check_read(batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd, out)
    if out is None:
        return _OP_READ(batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, dtype, hnd, pdl)
    key, value = out
    _OP_READ_OUT(key, value, batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd, pdl)
    return key, value


def _check_read(batch_indices, positions, k_codes, v_codes, pairs, kv_indices, kv_indptr, hnd, out) -> None:
    heads, head_dim = _check_cache(k_codes, v_codes, pairs, hnd)
    nnz = batch_indices.shape[0]
    _check_rows(batch_indices, positions, kv_indptr, nnz)
    key, value = (None, None) if out is None else out
    if out is not None:
        if tuple(key.shape) != (nnz, heads, head_dim) or value.shape != key.shape:
            raise ValueError(f"out must be two {(nnz, heads, head_dim)} tensors")
        if key.dtype != value.dtype:
            raise ValueError("out's tensors must share one dtype")
        _act_code(key)
        if key.stride(2) != 1 or value.stride(2) != 1:
            raise ValueError("out must be contiguous in head_dim")
    _check_device(k_codes, batch_indices=batch_indices, positions=positions, kv_indices=kv_indices, kv_indptr=kv_indptr,
                  key=key, value=value)


# ------------------------------------------------------------------------------------------------
# Attention.
# ------------------------------------------------------------------------------------------------
def paged_attention_int4(query: torch.Tensor, paged_kv_cache, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                         cum_seq_lens_q: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                         causal: bool = True, kv_layout: str = "NHD", out: Optional[torch.Tensor] = None,
                         return_lse: bool = False, enable_pdl: Optional[bool] = None):
    r"""``softmax(sm_scale * q k^T) v`` of ragged query rows over the 4-bit paged cache.

    `query` is ``(tokens, num_q_heads, head_dim)`` or ``(tokens, num_q_heads * head_dim)``, bfloat16 or float16, and may be a
    view of a qkv row; query head h reads kv head ``h // (num_q_heads // num_kv_heads)``. Request b's queries are rows
    ``cum_seq_lens_q[b]`` to ``cum_seq_lens_q[b + 1]`` (int32, ``(batch_size + 1,)``; None: one each, a decode step) and its
    keys the ``seq_lens[b]`` tokens that ``block_tables[b]`` lists, the queries' own appended. With `causal` query j of n sees
    the first ``seq_lens[b] - n + j + 1`` tokens; without, all. A query that sees none gives zeros; rows of `query` that no
    request covers are not written. Decode steps, drafts to verify and prompt chunks go through one call. All lengths stay on
    the device, so a captured call follows them.

    Keys and values enter the products as exact codes, with their scales applied in fp32; sums and softmax statistics
    are fp32, the weights of the value codes fp16 (relative to the row's largest), and the result is rounded once. Rows of very unlike
    scales may stand in one cache: values up to 2^90 in size, key rows of any finite size, queries below 2^123 (larger ones count as
    that large beside tiny keys). `sm_scale` defaults to ``head_dim ** -0.5``. With `return_lse`, returns
    ``(out, lse)``: fp32 ``(tokens, num_q_heads)``, the log2 of the summed exponentials (-inf for a query without keys), as the merging of
    partial attentions takes it. `out` may be `query` itself. A page id out of range reads as zeros and lengths that do not fit the table or
    `query` are cut to them; both set STATUS_KV_SLOT_OUT_OF_RANGE.
    """
    hnd = _is_hnd(kv_layout)
    k_codes, v_codes, pairs = _parts(paged_kv_cache)
    pdl = True if enable_pdl is None else bool(enable_pdl)
    if not query.is_cuda:
        _check_attention(query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, hnd, out)
    if out is None:
        out, lse = _OP_ATTENTION(query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, sm_scale, causal, hnd,
                                 return_lse, pdl)
    else:
        lse = None
        if return_lse:
            heads = query.shape[1] if query.dim() == 3 else query.shape[1] // (2 * k_codes.shape[3])
            lse = torch.empty((query.shape[0], heads), dtype=torch.float32, device=query.device)
        _OP_ATTENTION_OUT(out, lse, query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, sm_scale, causal,
                          hnd, pdl)
    return (out, lse) if return_lse else out


def _check_attention(query, k_codes, v_codes, pairs, block_tables, seq_lens, cum_seq_lens_q, hnd, out) -> None:
    kv_heads, head_dim = _check_cache(k_codes, v_codes, pairs, hnd)
    q = _heads(query, head_dim)
    _act_code(q)
    if q.shape[2] != head_dim or q.shape[1] == 0 or q.shape[1] % kv_heads:
        raise ValueError(f"query heads/head_dim {tuple(q.shape[1:])} do not go with the cache's {(kv_heads, head_dim)}")
    if q.stride(2) != 1:
        raise ValueError("query must be contiguous in head_dim")
    batch = _check_tables(block_tables, seq_lens)
    if cum_seq_lens_q is None:
        if q.shape[0] != batch:
            raise ValueError("without cum_seq_lens_q, query must have one row a request")
    else:
        _check_int32("cum_seq_lens_q", cum_seq_lens_q, (batch + 1,))
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.stride(-1) != 1):
        raise ValueError("out must have the shape and dtype of query and be contiguous in head_dim")
    _check_device(q, k_codes=k_codes, block_tables=block_tables, seq_lens=seq_lens, cum_seq_lens_q=cum_seq_lens_q, out=out)
