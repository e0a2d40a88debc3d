"""The paged KV cache in 4 bits: 4.25 bits an element in place of 16.

A head's row is held in blocks of 32 elements: 32 E2M1 codes (a sign and one of 0, 0.5,
1, 1.5, 2, 3, 4, 6) and the exponent of the block's power-of-two scale, the smallest
that keeps the largest magnitude within 6.  An element is off by at most a quarter of
its block's largest magnitude / 1.5 (half the step between 4 and 6, at a scale just past
a power of two), and by its block's scale / 4 where it is small.

``append_paged_kv_fp4`` writes tokens as ``append_paged_kv_batch`` does to a 16-bit
cache, ``gather_paged_kv_fp4`` reads the stored values back, and
``layers.paged_attention`` attends over the cache.  No counterpart in the reference,
whose page manager keeps a 16-bit cache (engine/page_manager.py:36-42).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .. import _lib


@dataclass
class Fp4KVCache:
    """One layer of the cache, [pages, 2, kv heads, page slots, ...], K at index 0.

    codes: uint8 [..., head_dim / 2], element 2 i in the low and 2 i + 1 in the high 4
    bits of byte i; scales: uint8 [..., head_dim / 32], 127 + the scale's exponent (255:
    the block reads as NaN)."""

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        c, s = self.codes, self.scales
        if c.dtype != torch.uint8 or s.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if c.dim() != 5 or s.dim() != 5 or c.shape[1] != 2 or c.shape[:4] != s.shape[:4] or c.shape[4] != 16 * s.shape[4]:
            raise ValueError(f"codes {tuple(c.shape)} and scales {tuple(s.shape)} must be "
                             "[pages, 2, heads, slots, head_dim / 2] and [pages, 2, heads, slots, head_dim / 32]")
        if c.stride(4) != 1 or s.stride(4) != 1:
            if c.shape[4] and (c.stride(4) != 1 or s.shape[4] > 1):
                raise ValueError("codes and scales must have unit stride along head_dim")

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

    @property
    def num_pages(self) -> int:
        return self.codes.shape[0]

    @property
    def num_kv_heads(self) -> int:
        return self.codes.shape[2]

    @property
    def page_size(self) -> int:
        return self.codes.shape[3]

    @property
    def head_dim(self) -> int:
        return 2 * self.codes.shape[4]


def _ints(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    if t.dim() != 1:
        raise ValueError(f"{name} must be one-dimensional")
    return t.contiguous()


def _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, num_tokens):
    """Checked token addressing: the tensors, which the call must keep, and their
    entry-point arguments."""
    positions, kv_indices = _ints("positions", positions), _ints("kv_indices", kv_indices)
    if positions.shape[0] != num_tokens:
        raise IndexError(f"{positions.shape[0]} positions for {num_tokens} tokens")
    if (kv_indptr is None) != (batch_indices is None):
        raise ValueError("kv_indptr and batch_indices go together")
    if kv_indptr is not None:
        batch_indices = _ints("batch_indices", batch_indices)
        if batch_indices.shape[0] != num_tokens:
            raise IndexError(f"{batch_indices.shape[0]} batch indices for {num_tokens} tokens")
        if kv_indptr.dtype != torch.int32 or kv_indptr.dim() != 1 or kv_indptr.shape[0] < 1:
            raise TypeError("kv_indptr must be a one-dimensional int32 tensor")
        kv_indptr = kv_indptr.contiguous()
    if cache.page_size == 0 and num_tokens:
        raise ValueError("the cache's pages have no slots")
    keep = (positions, kv_indices, kv_indptr, batch_indices)
    args = (kv_indices.data_ptr(), _lib.dtype_code(kv_indices), kv_indices.shape[0], _lib.ptr(kv_indptr),
            _lib.ptr(batch_indices), _lib.dtype_code(batch_indices) if batch_indices is not None else 0,
            kv_indptr.shape[0] - 1 if kv_indptr is not None else 0, positions.data_ptr(), _lib.dtype_code(positions))
    return keep, args


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
    for name, t in (("k", k), ("v", v)):
        if tuple(t.shape) != (tokens, heads, dim):
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not match the cache's [tokens, {heads}, {dim}] rows")
    if k.dtype != v.dtype:
        raise TypeError(f"k and v must share a dtype (got {k.dtype} and {v.dtype})")
    code = _lib.dtype_code(k)
    if code > _lib.BF16:
        raise TypeError(f"k and v must be bf16, fp16 or fp32, not {k.dtype}")
    k = k if k.stride(2) == 1 else k.contiguous()
    v = v if v.stride(2) == 1 else v.contiguous()
    keep, where = _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, tokens)
    dev = _lib.require_device(k, v, cache.codes, cache.scales, *keep)
    if tokens == 0:
        return
    with _lib.on_device(dev):
        _lib.call("bfa_append_paged_kv_fp4", k.data_ptr(), v.data_ptr(), code, tokens, heads, dim,
                  k.stride(0), k.stride(1), v.stride(0), v.stride(1), cache.codes.data_ptr(), cache.scales.data_ptr(),
                  cache.num_pages, cache.page_size, *cache.codes.stride()[:4], *cache.scales.stride()[:4], *where,
                  _lib.status_word(dev).data_ptr(), _lib.stream_of(dev))


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
    code = _lib.dtype_code(dtype)
    if code > _lib.BF16:
        raise TypeError(f"dtype must be bf16, fp16 or fp32, not {dtype}")
    tokens, heads, dim = positions.shape[0], cache.num_kv_heads, cache.head_dim
    keep, where = _tokens(cache, kv_indices, kv_indptr, batch_indices, positions, tokens)
    dev = _lib.require_device(cache.codes, cache.scales, *keep)
    k, v = (torch.empty(tokens, heads, dim, dtype=dtype, device=dev) for _ in range(2))
    if tokens == 0:
        return k, v
    with _lib.on_device(dev):
        _lib.call("bfa_gather_paged_kv_fp4", cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_pages,
                  cache.page_size, heads, dim, *cache.codes.stride()[:4], *cache.scales.stride()[:4], *where, tokens,
                  k.data_ptr(), v.data_ptr(), code, _lib.status_word(dev).data_ptr(), _lib.stream_of(dev))
    return k, v
