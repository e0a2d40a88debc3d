"""A step's batch of requests, built on the GPU from their lengths.

``build_paged_kv_indices`` (kernels/kv_cache_utils.py) walks Python lists and copies
three tensors to the device; an engine whose lengths change every step (and are known
on the device first, after sampling or after drafts were accepted) builds the same
CSR page lists, and each new token's position and cache slot, in one launch of
``bfa_build_paged_kv_batch`` here.  What it returns is what ``append_paged_kv_batch``,
``append_paged_kv_fp4``, ``qk_norm_rope`` and ``paged_attention`` take.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib


class PagedKVBatch(NamedTuple):
    """A step's batch; what is behind the last request holds -1."""

    qo_indptr: torch.Tensor         # [B + 1] int32: request b's new tokens are qo_indptr[b]:qo_indptr[b + 1]
    kv_indptr: torch.Tensor         # [B + 1] int32: its pages are kv_indices[kv_indptr[b]:kv_indptr[b + 1]]
    kv_indices: torch.Tensor        # [page_tables.numel()] int32
    kv_last_page_len: torch.Tensor  # [B] int32: tokens on its last page
    batch_indices: torch.Tensor     # [num_tokens] int32: each new token's request
    positions: torch.Tensor         # [num_tokens] int64: its position
    slot_mapping: torch.Tensor      # [num_tokens] int64: its page id * page_size + slot on the page


_DTYPES = (torch.int32, torch.int32, torch.int32, torch.int32, torch.int32, torch.int64, torch.int64)
_INTS = {torch.int32: _lib.I32, torch.int64: _lib.I64}


def build_paged_kv_batch(
    page_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    query_lens: torch.Tensor,
    page_size: int,
    num_tokens: int,
    out: Optional[PagedKVBatch] = None,
) -> PagedKVBatch:
    """page_tables [B, max_pages], seq_lens [B] (tokens in the cache after the step) and
    query_lens [B] (the new ones among them), int32 or int64 on the device.

    num_tokens: rows of the step's token tensors, at least the sum of query_lens; a
    padded batch (a captured graph's) has more.  out: tensors of an earlier call of
    the same sizes, written again.  Nothing is read back: lengths that do not fit
    raise IndexError at the next ``braidinfer_amd.check_device_status()``.  For an
    append of a padded batch pass the live tokens' slices to ``append_paged_kv_batch``
    (it takes request -1 for an error); ``append_paged_kv_fp4`` skips padding itself.
    """
    if page_tables.dim() != 2:
        raise ValueError("page_tables must be [requests, max_pages]")
    seqs, width = page_tables.shape
    codes = []
    for name, t, dims in (("seq_lens", seq_lens, 1), ("query_lens", query_lens, 1), ("page_tables", page_tables, 2)):
        if t.dim() != dims or t.shape[0] != seqs:
            raise ValueError(f"{name} of shape {tuple(t.shape)} for {seqs} requests")
        code = _INTS.get(t.dtype)
        if code is None:
            raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
        codes.append(code)
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    if width and page_tables.stride(1) != 1:
        page_tables = page_tables.contiguous()
    seq_lens, query_lens = seq_lens.contiguous(), query_lens.contiguous()
    dev = _lib.require_device(page_tables, seq_lens, query_lens)
    sizes = (seqs + 1, seqs + 1, seqs * width, seqs, num_tokens, num_tokens, num_tokens)
    if out is None:
        # two allocations for the seven (one of 1.4 us each otherwise)
        out = PagedKVBatch(*torch.empty(sum(sizes[:5]), dtype=torch.int32, device=dev).split_with_sizes(sizes[:5]),
                           *torch.empty(2, num_tokens, dtype=torch.int64, device=dev).unbind())
    else:
        for name, t, n, d in zip(out._fields, out, sizes, _DTYPES):
            if t.dtype != d or tuple(t.shape) != (n,) or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous {d} tensor of {n} elements")
        _lib.require_device(page_tables, *out)
    with _lib.on_device(dev):
        rc = _lib.entry("bfa_build_paged_kv_batch")(
            page_tables.data_ptr(), codes[2], seqs, width, page_tables.stride(0), seq_lens.data_ptr(), codes[0],
            query_lens.data_ptr(), codes[1], int(page_size), num_tokens, seqs * width, *[t.data_ptr() for t in out],
            _lib.status_word(dev).data_ptr(), _lib.stream_of(dev))
    if rc < 0:
        _lib.raise_error(rc)
    return out
