"""The paged KV cache in 4 bits: 4.25 bits an element in place of 16.

A head's row is held in blocks of 32 elements: 32 E2M1 codes (a sign and one of 0, 0.5,
1, 1.5, 2, 3, 4, 6) and the exponent of the block's power-of-two scale, the smallest
that keeps the largest magnitude within 6.  An element is off by at most half a step of
its magnitude's range: a quarter of the scale up to 2 scales, half of it up to 4, and all
of it up to 6, which is at most a fifth of the block's largest magnitude.

``append_paged_kv_fp4`` writes tokens as ``append_paged_kv_batch`` does to a 16-bit
cache, ``gather_paged_kv_fp4`` reads the stored values back, and
``layers.paged_attention`` attends over the cache.  No counterpart in the reference,
whose page manager keeps a 16-bit cache (engine/page_manager.py:36-42).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib


class Fp4KVCache:
    """One layer of the cache, [pages, 2, kv heads, page slots, ...], K at index 0.

    codes: uint8 [..., head_dim / 2], element 2 i in the low and 2 i + 1 in the high 4
    bits of byte i; scales: uint8 [..., head_dim / 32], 127 + the scale's exponent (255:
    the block reads as NaN)."""

    __slots__ = ("codes", "scales", "num_pages", "num_kv_heads", "page_size", "head_dim", "strides")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        c, s = codes.shape, scales.shape
        if len(c) != 5 or len(s) != 5 or c[1] != 2 or c[:4] != s[:4] or c[4] != 16 * s[4]:
            raise ValueError(f"codes {tuple(c)} and scales {tuple(s)} must be "
                             "[pages, 2, heads, slots, head_dim / 2] and [pages, 2, heads, slots, head_dim / 32]")
        cs, ss = codes.stride(), scales.stride()
        if (cs[4] != 1 and c[4] > 1) or (ss[4] != 1 and s[4] > 1):
            raise ValueError("codes and scales must have unit stride along head_dim")
        pages, _, heads, slots, half = c
        strides = cs[:4] + ss[:4]  # (page, K|V, head, slot) of the codes and of the scales, in bytes
        for name, value in zip(self.__slots__, (codes, scales, pages, heads, slots, 2 * half, strides)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{name} of an Fp4KVCache stays as it is: make another of the new tensors")

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device=None) -> "Fp4KVCache":
        """A cache that holds no tokens yet (its memory is not cleared)."""
        if head_dim <= 0 or head_dim % 32:
            raise ValueError(f"head_dim {head_dim} (a multiple of 32)")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        shape = (num_pages, 2, num_kv_heads, page_size)
        return cls(torch.empty(*shape, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.empty(*shape, head_dim // 32, dtype=torch.uint8, device=device))


_INTS = {torch.int32: _lib.I32, torch.int64: _lib.I64}
_FLOATS = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _ints(name: str, t: torch.Tensor, n=None):
    """(contiguous one-dimensional int32 or int64 tensor, of n elements if given; its code)"""
    code = _INTS.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    shape = t.shape
    if len(shape) != 1:
        raise ValueError(f"{name} must be one-dimensional")
    if n is not None and shape[0] != n:
        raise IndexError(f"{shape[0]} {name.replace('_', ' ')} for {n} tokens")
    return (t if t.is_contiguous() else t.contiguous()), code


def _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, num_tokens):
    """Checked token addressing: the tensors, which the call must keep, and their
    entry-point arguments."""
    positions, pos_code = _ints("positions", positions, num_tokens)
    kv_indices, idx_code = _ints("kv_indices", kv_indices)
    if cache.page_size == 0 and num_tokens:
        raise ValueError("the cache's pages have no slots")
    if kv_indptr is None and batch_indices is None:
        return (positions, kv_indices, None, None), (kv_indices.data_ptr(), idx_code, kv_indices.shape[0], None, None, 0, 0,
                                                     positions.data_ptr(), pos_code)
    if kv_indptr is None or batch_indices is None:
        raise ValueError("kv_indptr and batch_indices go together")
    batch_indices, code = _ints("batch_indices", batch_indices, num_tokens)
    shape = kv_indptr.shape
    if kv_indptr.dtype != torch.int32 or len(shape) != 1 or shape[0] < 1:
        raise TypeError("kv_indptr must be a one-dimensional int32 tensor")
    if not kv_indptr.is_contiguous():
        kv_indptr = kv_indptr.contiguous()
    return (positions, kv_indices, kv_indptr, batch_indices), (
        kv_indices.data_ptr(), idx_code, kv_indices.shape[0], kv_indptr.data_ptr(), batch_indices.data_ptr(), code,
        shape[0] - 1, positions.data_ptr(), pos_code)


def append_paged_kv_fp4(
    k: torch.Tensor,
    v: torch.Tensor,
    cache: Fp4KVCache,
    kv_indices: torch.Tensor,
    kv_indptr: Optional[torch.Tensor],
    batch_indices: Optional[torch.Tensor],
    positions: torch.Tensor,
) -> None:
    """Writes token t's K and V (``k[t]``, ``v[t]``: [kv heads, head_dim], bf16, fp16 or
    fp32) at ``positions[t]`` of request ``batch_indices[t]``, whose pages are
    ``kv_indices[kv_indptr[b]:kv_indptr[b + 1]]``; without kv_indptr and batch_indices
    all of kv_indices is one request's.  A token of request -1 (the padding of
    ``build_paged_kv_batch``) is skipped; one past its page list is skipped and warned
    of, and other out-of-range indices raise IndexError, at the next
    ``braidinfer_amd.check_device_status()``.  Tokens must have distinct slots."""
    tokens, heads, dim = k.shape[0], cache.num_kv_heads, cache.head_dim
    shape = (tokens, heads, dim)
    if k.shape != shape or v.shape != shape:
        name, t = ("k", k) if k.shape != shape else ("v", v)
        raise ValueError(f"{name} of shape {tuple(t.shape)} does not match the cache's [tokens, {heads}, {dim}] rows")
    if k.dtype != v.dtype:
        raise TypeError(f"k and v must share a dtype (got {k.dtype} and {v.dtype})")
    code = _FLOATS.get(k.dtype)
    if code is None:
        raise TypeError(f"k and v must be bf16, fp16 or fp32, not {k.dtype}")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        k, v = k.contiguous(), v.contiguous()
        ks, vs = k.stride(), v.stride()
    keep, where = _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, tokens)
    dev = _lib.require_device(k, v, cache.codes, cache.scales, *keep)
    if tokens == 0:
        return
    _lib.launch(_lib.entry("bfa_append_paged_kv_fp4"), dev, k.data_ptr(), v.data_ptr(), code, tokens, heads, dim, ks[0],
                ks[1], vs[0], vs[1], cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_pages, cache.page_size,
                *cache.strides, *where)


def gather_paged_kv_fp4(
    cache: Fp4KVCache,
    kv_indices: torch.Tensor,
    kv_indptr: Optional[torch.Tensor],
    batch_indices: Optional[torch.Tensor],
    positions: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(K, V), each [tokens, kv heads, head_dim] in `dtype`: the values the cache holds
    for the tokens addressed as in ``append_paged_kv_fp4`` (to move cached tokens to a
    16-bit cache, or to compare with what was stored).  bf16 and fp32 hold every value
    exactly, but for 2^128, to which magnitudes from 3.5 x 2^126 round: it reads as
    infinity, and in fp16 so does all that is past its range.  A token without a place, and padding, reads as zeros."""
    code = _FLOATS.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, not {dtype}")
    tokens, heads, dim = positions.shape[0], cache.num_kv_heads, cache.head_dim
    keep, where = _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, tokens)
    dev = _lib.require_device(cache.codes, cache.scales, *keep)
    k, v = torch.empty((2, tokens, heads, dim), dtype=dtype, device=dev).unbind()
    if tokens == 0:
        return k, v
    _lib.launch(_lib.entry("bfa_gather_paged_kv_fp4"), dev, cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_pages,
                cache.page_size, heads, dim, *cache.strides, *where, tokens, k.data_ptr(), v.data_ptr(), code)
    return k, v
