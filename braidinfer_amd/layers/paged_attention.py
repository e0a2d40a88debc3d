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


def _aligned(t: torch.Tensor, unit: int) -> bool:
    """16-byte aligned, with strides (but the last, which is 1) in multiples of `unit`."""
    st = t.stride()
    return st[-1] == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s, n in zip(st[:-1], t.shape) if n > 1)


def _strides(t: torch.Tensor, dims) -> list[int]:
    """Strides along `dims`, 0 for a dimension of one element (whose stride means nothing)."""
    st = t.stride()
    return [st[i] if t.shape[i] > 1 else 0 for i in dims]


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
    code = _lib.dtype_code(query)
    if code not in (_lib.BF16, _lib.F16):
        raise TypeError(f"query must be bf16 or fp16, not {query.dtype}")
    if isinstance(kv_cache, Fp4KVCache):
        data, scales, cache_code = kv_cache.codes, kv_cache.scales, _lib.FP4
        if kv_layout != "HND":
            raise ValueError("a 4-bit cache has layout HND")
        pages, hkv, slots, cache_dim = kv_cache.num_pages, kv_cache.num_kv_heads, kv_cache.page_size, kv_cache.head_dim
        st, sst = _strides(data, (0, 1, 2, 3)), _strides(scales, (0, 1, 2, 3))
        unit = 16
    else:
        if kv_layout not in _LAYOUT_DIMS:
            raise ValueError(f"Unknown kv_layout: {kv_layout}")
        if kv_cache.dim() != 5 or kv_cache.shape[1] != 2:
            raise ValueError("kv_cache must be one layer [num_pages, 2, ...] with 5 dimensions")
        if kv_cache.dtype != query.dtype:
            raise TypeError(f"query and kv_cache must share a dtype (got {query.dtype} and {kv_cache.dtype})")
        h, s = _LAYOUT_DIMS[kv_layout]
        data, scales, cache_code = kv_cache, None, code
        pages, hkv, slots, cache_dim = kv_cache.shape[0], kv_cache.shape[h], kv_cache.shape[s], kv_cache.shape[4]
        st, sst = _strides(data, (0, 1, h, s)), (0, 0, 0, 0)
        unit = 8
    if cache_dim != dim:
        raise ValueError(f"kv_cache holds rows of {cache_dim} elements, query of {dim}")
    if dim not in (64, 128):
        raise ValueError(f"head_dim {dim} (64 or 128)")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"{hq} query heads do not share {hkv} kv heads evenly")
    if slots == 0:
        raise ValueError("the cache's pages have no slots")
    if pages and not _aligned(data, unit):
        raise ValueError("kv_cache must be 16-byte aligned, with unit stride along head_dim and others in multiples of 16 bytes")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1 (None for no window)")
    if num_sinks < 0:
        raise ValueError("num_sinks must not be negative")
    seqs = kv_last_page_len.shape[0] if kv_last_page_len.dim() == 1 else -1
    lists = []
    for name, t, n in (("kv_indices", kv_indices, None), ("kv_indptr", kv_indptr, seqs + 1),
                       ("kv_last_page_len", kv_last_page_len, seqs), ("qo_indptr", qo_indptr, seqs + 1)):
        if t.dtype != torch.int32 or t.dim() != 1:
            raise TypeError(f"{name} must be a one-dimensional int32 tensor")
        if n is not None and t.shape[0] != n:
            raise ValueError(f"{name} has {t.shape[0]} elements, for {seqs} requests {n} are needed")
        lists.append(t if t.is_contiguous() else t.contiguous())
    kv_indices, kv_indptr, kv_last_page_len, qo_indptr = lists
    if not _aligned(query, 8):
        query = query.contiguous()
        if query.data_ptr() % 16:
            query = query.clone()
    dev = _lib.require_device(query, data, scales, *lists, out)
    if out is None:
        out = torch.empty(tokens, hq * dim, dtype=query.dtype, device=dev)
    elif out.dtype != query.dtype or tuple(out.shape) != (tokens, hq * dim) or not _aligned(out, 8):
        raise ValueError(f"out must be a 16-byte aligned [{tokens}, {hq * dim}] tensor of the query's dtype, its row "
                         "stride a multiple of 8")
    if tokens == 0 or seqs == 0:
        return out
    win = 0 if window is None else int(window)
    size = _lib.workspace_size("bfa_paged_attention_workspace_size", tokens, seqs, hq, hkv, dim, kv_indices.shape[0], slots,
                               win, int(num_sinks), cache_code)
    qs = _strides(query, (0, 1))
    ws = _lib.scratch(dev)
    with _lib.on_device(dev), ws.lock:
        ws.reserve(size)
        _lib.call("bfa_paged_attention", query.data_ptr(), code, tokens, hq, qs[0], qs[1], data.data_ptr(), cache_code,
                  pages, hkv, slots, dim, *st, _lib.ptr(scales), *sst, kv_indices.data_ptr(), kv_indices.shape[0],
                  kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), qo_indptr.data_ptr(), seqs,
                  dim ** -0.5 if scale is None else float(scale), win, int(num_sinks), out.data_ptr(),
                  out.stride(0) if tokens > 1 else hq * dim, ws.ptr, ws.size, _lib.status_word(dev).data_ptr(),
                  _lib.stream_of(dev))
    return out
