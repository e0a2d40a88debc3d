"""RMSNorm of query and key heads with their rotation, in one pass, on MI355X.

``qwen3_attention_input`` has both in the epilogue of its QKV projection.  A q and k
that come from another projection (``QKVParallelLinear.forward``, ``linear``) take
``q_norm``, ``k_norm`` and ``rotary_emb`` one after the other in the reference
(models/qwen3.py:257-309), three launches that read and write them twice; here it is
one.  The arithmetic is fp32 and rounded once, where the three calls round the normed
heads to the tensors' dtype in between.
"""
from __future__ import annotations

import torch

from .. import _lib


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    q_norm_weight: torch.Tensor | None,
    k_norm_weight: torch.Tensor | None,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """New tensors of query's and key's shapes: each head's row normed with its weight
    (None: not normed), then rotated by the token's position.

    query, key: [T, heads * head_dim] or [T, heads, head_dim] views of one dtype (bf16,
    fp16 or fp32), which may be slices of a packed projection; head_dim is that of
    cos_sin_cache (fp32 [max_position, head_dim], as ``RotaryEmbedding`` holds it),
    even.  positions [T], int32 or int64; as torch indexing takes them, with positions
    out of range raised by ``braidinfer_amd.check_device_status()``."""
    if cos_sin_cache.dim() != 2 or cos_sin_cache.dtype != torch.float32:
        raise ValueError("cos_sin_cache must be float32 [max_position, head_dim]")
    max_position, dim = cos_sin_cache.shape
    pos_code = _INTS.get(positions.dtype)
    if pos_code is None or positions.dim() != 1:
        raise ValueError("positions must be a one-dimensional int32 or int64 tensor")
    tokens = positions.shape[0]
    if dim == 0 or dim % 2:
        raise ValueError(f"head_dim {dim} must be even")
    if query.dtype != key.dtype:
        raise TypeError(f"query and key must share a dtype (got {query.dtype} and {key.dtype})")
    code = _FLOATS.get(query.dtype)
    if code is None:
        raise TypeError(f"query and key must be bf16, fp16 or fp32, not {query.dtype}")
    q, q_heads, q_token, q_head = _rows("query", query, tokens, dim)
    k, k_heads, k_token, k_head = _rows("key", key, tokens, dim)
    qw, qw_ptr, w_code = _weight(q_norm_weight, dim)
    kw, kw_ptr, k_code = _weight(k_norm_weight, dim)
    if k_code != w_code:
        if qw is not None and kw is not None:
            raise TypeError("norm weights must share a dtype: bf16, fp16 or fp32")
        w_code = w_code if kw is None else k_code
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if not cos_sin_cache.is_contiguous():
        cos_sin_cache = cos_sin_cache.contiguous()
    dev = _lib.require_device(q, k, positions, cos_sin_cache, qw, kw)
    q_out = torch.empty(query.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(key.shape, dtype=q.dtype, device=dev)
    if tokens:
        _lib.launch(_lib.entry("bfa_qk_norm_rope"), dev, q.data_ptr(), q_heads, q_token, q_head, q_out.data_ptr(),
                    k.data_ptr(), k_heads, k_token, k_head, k_out.data_ptr(), code, tokens, dim, qw_ptr, kw_ptr, w_code, eps,
                    positions.data_ptr(), pos_code, cos_sin_cache.data_ptr(), max_position)
    return q_out, k_out


def _weight(w: torch.Tensor | None, dim: int):
    """(contiguous weight, its address, its dtype's code)"""
    if w is None:
        return None, None, 0
    if w.numel() != dim:
        raise ValueError(f"norm weights must have head_dim = {dim} elements")
    code = _FLOATS.get(w.dtype)
    if code is None:
        raise TypeError("norm weights must share a dtype: bf16, fp16 or fp32")
    if not w.is_contiguous():
        w = w.detach().contiguous()
    return w, w.data_ptr(), code


_INTS = {torch.int32: _lib.I32, torch.int64: _lib.I64}
_FLOATS = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _rows(name: str, x: torch.Tensor, tokens: int, dim: int):
    """(x with unit stride along a head's row, heads, token stride, head stride)"""
    shape = x.shape
    if len(shape) == 2 and shape[0] == tokens and shape[1] % dim == 0:
        token, last = x.stride()
        if last != 1:
            x = x.contiguous()
            token = shape[1]
        return x, shape[1] // dim, token, dim
    if len(shape) == 3 and shape[0] == tokens and shape[2] == dim:
        if x.stride(2) != 1:
            x = x.contiguous()
        token, head, _ = x.stride()
        return x, shape[1], token, head
    raise ValueError(f"{name} of shape {tuple(shape)} is not [{tokens}, heads * {dim}] or [{tokens}, heads, {dim}]")
