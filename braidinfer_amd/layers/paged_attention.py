"""Causal attention of a batch of requests over one paged cache, on MI355X.

``CascadeAttention`` serves one stream of tokens over chunks that it shares with
others; a batch of independent requests, each with its own pages, is one call here
(``bfa_paged_attention``): any mix of single new tokens and pieces of prompts, over a
16-bit cache or a 4-bit one (``kernels.Fp4KVCache``), with an optional sliding window
and first tokens ("sinks") that stay visible behind it.  The page lists are those of
``build_paged_kv_indices`` or, built on the device, ``build_paged_kv_batch``.
"""
from __future__ import annotations

import torch

from .. import _lib
from ..kernels.fp4_kv_cache import Fp4KVCache

_LAYOUT_DIMS = {"HND": (2, 3), "NHD": (3, 2)}  # (head dim, slot dim) of the 5-D layer cache


_QUERY = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _strides(t: torch.Tensor, unit: int):
    """Strides of t, multiples of `unit` but for the last, which is 1, and 16-byte
    aligned; None if they are not.  0 for a dimension of one element, whose stride means
    nothing, where it is not such a multiple."""
    st = t.stride()
    if (st[0] | st[1] | (0 if len(st) < 4 else st[2] | st[3])) % unit:
        st = tuple(0 if n == 1 else s for n, s in zip(t.shape[:-1], st)) + st[-1:]
        if any(s % unit for s in st[:-1]):
            return None
    return st if st[-1] == 1 and t.data_ptr() % 16 == 0 else None


def paged_attention(
    query: torch.Tensor,
    kv_cache: torch.Tensor | Fp4KVCache,
    kv_indices: torch.Tensor,
    kv_indptr: torch.Tensor,
    kv_last_page_len: torch.Tensor,
    qo_indptr: torch.Tensor,
    scale: float | None = None,
    window: int | None = None,
    num_sinks: int = 0,
    kv_layout: str = "HND",
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """[T, Hq * head_dim]: request s's query rows ``qo_indptr[s]:qo_indptr[s + 1]`` attend
    its cached tokens, which must already hold the rows' own keys and values.

    query: [T, Hq, head_dim], bf16 or fp16, head_dim 64 or 128.  kv_cache: one layer, of
    the query's dtype ([pages, 2, Hkv, slots, head_dim] "HND", [pages, 2, slots, Hkv,
    head_dim] "NHD"), or an Fp4KVCache.  kv_indices, kv_indptr, kv_last_page_len,
    qo_indptr: int32; the request's tokens fill its pages in order, the last one with
    kv_last_page_len.  Its rows are its last tokens: the last row sees every key, each
    earlier one a key less.  With ``window``, a row sees the last ``window`` keys, its
    own the last of them, and the first ``num_sinks`` of the request.  scale: of the
    scores, head_dim ** -0.5 unless given.

    A row that sees no key (a request without pages) is 0.  Rows of ``out`` past the
    last request are left as they were (uninitialised without ``out``).  Page ids that
    do not exist and offsets outside the tensors raise IndexError at the next
    ``braidinfer_amd.check_device_status()``.  Scratch memory: see
    ``braidinfer_amd._lib.scratch``."""
    if query.dim() != 3:
        raise ValueError(f"query of shape {tuple(query.shape)} is not [tokens, heads, head_dim]")
    tokens, hq, dim = query.shape
    dtype = query.dtype
    code = _QUERY.get(dtype)
    if code is None:
        raise TypeError(f"query must be bf16 or fp16, not {dtype}")
    if isinstance(kv_cache, Fp4KVCache):
        if kv_layout != "HND":
            raise ValueError("a 4-bit cache has layout HND")
        data, scales, cache_code, unit = kv_cache.codes, kv_cache.scales, _lib.FP4, 16
        pages, hkv, slots, cache_dim = kv_cache.num_pages, kv_cache.num_kv_heads, kv_cache.page_size, kv_cache.head_dim
        h, s = 2, 3
        sst = kv_cache.strides[4:]
    else:
        dims = _LAYOUT_DIMS.get(kv_layout)
        if dims is None:
            raise ValueError(f"Unknown kv_layout: {kv_layout}")
        h, s = dims
        data, scales, cache_code, unit = kv_cache, None, code, 8
        shape = data.shape
        if len(shape) != 5 or shape[1] != 2:
            raise ValueError("kv_cache must be one layer [num_pages, 2, ...] with 5 dimensions")
        if data.dtype != dtype:
            raise TypeError(f"query and kv_cache must share a dtype (got {dtype} and {data.dtype})")
        pages, hkv, slots, cache_dim = shape[0], shape[h], shape[s], shape[4]
        sst = (0, 0, 0, 0)
    if cache_dim != dim:
        raise ValueError(f"kv_cache holds rows of {cache_dim} elements, query of {dim}")
    if dim not in (64, 128):
        raise ValueError(f"head_dim {dim} (64 or 128)")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"{hq} query heads do not share {hkv} kv heads evenly")
    if slots == 0:
        raise ValueError("the cache's pages have no slots")
    st = _strides(data, unit)
    if st is None:
        if pages:
            raise ValueError("kv_cache must be 16-byte aligned, with unit stride along head_dim and others in multiples of "
                             "16 bytes")
        st = (0, 0, 0, 0)
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError("window must be at least 1 (None for no window)")
    if num_sinks < 0:
        raise ValueError("num_sinks must not be negative")
    indices_shape, requests = kv_indices.shape, kv_last_page_len.shape
    i32 = torch.int32
    if (kv_indices.dtype != i32 or kv_indptr.dtype != i32 or kv_last_page_len.dtype != i32 or qo_indptr.dtype != i32
            or len(indices_shape) != 1 or len(requests) != 1):
        raise TypeError("kv_indices, kv_indptr, kv_last_page_len and qo_indptr must be one-dimensional int32 tensors")
    seqs, num_indices = requests[0], indices_shape[0]
    ends = (seqs + 1,)
    if kv_indptr.shape != ends or qo_indptr.shape != ends:
        name, t = ("kv_indptr", kv_indptr) if kv_indptr.shape != ends else ("qo_indptr", qo_indptr)
        raise ValueError(f"{name} has shape {tuple(t.shape)}, for {seqs} requests {seqs + 1} elements are needed")
    if not (kv_indices.is_contiguous() and kv_indptr.is_contiguous() and kv_last_page_len.is_contiguous()
            and qo_indptr.is_contiguous()):
        kv_indices, kv_indptr = kv_indices.contiguous(), kv_indptr.contiguous()
        kv_last_page_len, qo_indptr = kv_last_page_len.contiguous(), qo_indptr.contiguous()
    qs = _strides(query, 8)
    if qs is None:
        query = query.clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    dev = _lib.require_device(query, data, scales, kv_indices, kv_indptr, kv_last_page_len, qo_indptr, out)
    row = hq * dim
    if out is None:
        out = torch.empty((tokens, row), dtype=dtype, device=dev)
    else:
        ost = _strides(out, 8) if out.dtype == dtype and tuple(out.shape) == (tokens, row) else None
        if ost is None:
            raise ValueError(f"out must be a 16-byte aligned [{tokens}, {row}] tensor of the query's dtype, its row stride a "
                             "multiple of 8")
        row = ost[0]
    if tokens == 0 or seqs == 0:
        return out
    size = _lib.entry("bfa_paged_attention_workspace_size")(tokens, seqs, hq, hkv, dim, num_indices, slots, window, num_sinks,
                                                            cache_code)
    ws = _lib.scratch(dev)
    with ws.lock:
        if ws.size < size or ws.buf is None:
            ws.reserve(size)
        _lib.launch(_lib.entry("bfa_paged_attention"), dev, query.data_ptr(), code, tokens, hq, qs[0], qs[1], data.data_ptr(),
                    cache_code, pages, hkv, slots, dim, st[0], st[1], st[h], st[s],
                    None if scales is None else scales.data_ptr(), *sst, kv_indices.data_ptr(), num_indices,
                    kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), qo_indptr.data_ptr(), seqs,
                    dim ** -0.5 if scale is None else scale, window, num_sinks, out.data_ptr(), row, ws.ptr, ws.size)
    return out
