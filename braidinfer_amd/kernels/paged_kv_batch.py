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
    shape = page_tables.shape
    if len(shape) != 2:
        raise ValueError("page_tables must be [requests, max_pages]")
    seqs, width = shape
    if seq_lens.shape != (seqs,) or query_lens.shape != (seqs,):
        name, t = ("seq_lens", seq_lens) if seq_lens.shape != (seqs,) else ("query_lens", query_lens)
        raise ValueError(f"{name} of shape {tuple(t.shape)} for {seqs} requests")
    table_code, seq_code, query_code = _INTS.get(page_tables.dtype), _INTS.get(seq_lens.dtype), _INTS.get(query_lens.dtype)
    if table_code is None or seq_code is None or query_code is None:
        raise TypeError("page_tables, seq_lens and query_lens must be int32 or int64 "
                        f"(got {page_tables.dtype}, {seq_lens.dtype} and {query_lens.dtype})")
    if page_size <= 0:
        raise ValueError("page_size must be positive")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    row, column = page_tables.stride()
    if column != 1 and width:
        page_tables = page_tables.contiguous()
        row = width
    if not seq_lens.is_contiguous():
        seq_lens = seq_lens.contiguous()
    if not query_lens.is_contiguous():
        query_lens = query_lens.contiguous()
    dev = _lib.require_device(page_tables, seq_lens, query_lens)
    entries = seqs * width
    if out is None:
        # two allocations for the seven tensors
        words = torch.empty(2 * seqs + 2 + entries + seqs + num_tokens, dtype=torch.int32, device=dev)
        qo, kv, idx, last, owner = words.split_with_sizes((seqs + 1, seqs + 1, entries, seqs, num_tokens))
        positions, slots = torch.empty((2, num_tokens), dtype=torch.int64, device=dev).unbind()
        out = PagedKVBatch(qo, kv, idx, last, owner, positions, slots)
    else:
        sizes = (seqs + 1, seqs + 1, entries, seqs, num_tokens, num_tokens, num_tokens)
        for name, t, n, d in zip(out._fields, out, sizes, _DTYPES):
            if t.dtype != d or tuple(t.shape) != (n,) or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous {d} tensor of {n} elements")
        _lib.require_device(page_tables, *out)
        qo, kv, idx, last, owner, positions, slots = out
    _lib.launch(_lib.entry("bfa_build_paged_kv_batch"), dev, page_tables.data_ptr(), table_code, seqs, width, row,
                seq_lens.data_ptr(), seq_code, query_lens.data_ptr(), query_code, page_size, num_tokens, entries,
                qo.data_ptr(), kv.data_ptr(), idx.data_ptr(), last.data_ptr(), owner.data_ptr(), positions.data_ptr(),
                slots.data_ptr())
    return out
