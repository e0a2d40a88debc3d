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
    tokens = positions.shape[0] if positions.dim() == 1 else -1
    if tokens < 0 or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be a one-dimensional int32 or int64 tensor")
    if dim == 0 or dim % 2:
        raise ValueError(f"head_dim {dim} must be even")
    rows = []
    for name, x in (("query", query), ("key", key)):
        if x.dim() == 2 and x.shape[0] == tokens and x.shape[1] % dim == 0:
            rows.append((x if x.stride(1) == 1 else x.contiguous()).unflatten(1, (-1, dim)))
        elif x.dim() == 3 and x.shape[0] == tokens and x.shape[2] == dim:
            rows.append(x if x.stride(2) == 1 else x.contiguous())
        else:
            raise ValueError(f"{name} of shape {tuple(x.shape)} is not [{tokens}, heads * {dim}] or [{tokens}, heads, {dim}]")
    q, k = rows
    if q.dtype != k.dtype:
        raise TypeError(f"query and key must share a dtype (got {q.dtype} and {k.dtype})")
    code = _lib.dtype_code(q)
    if code > _lib.BF16:
        raise TypeError(f"query and key must be bf16, fp16 or fp32, not {q.dtype}")
    weights = [w.detach().contiguous() if w is not None else None for w in (q_norm_weight, k_norm_weight)]
    given = [w for w in weights if w is not None]
    w_code = _lib.F32
    if given:
        if any(w.numel() != dim for w in given):
            raise ValueError(f"norm weights must have head_dim = {dim} elements")
        w_code = _lib.dtype_code(given[0])
        if given[0].dtype != given[-1].dtype or w_code > _lib.BF16:
            raise TypeError("norm weights must share a dtype: bf16, fp16 or fp32")
    positions, cos_sin_cache = positions.contiguous(), cos_sin_cache.contiguous()
    dev = _lib.require_device(q, k, positions, cos_sin_cache, *given)
    q_out = torch.empty(query.shape, dtype=q.dtype, device=dev)
    k_out = torch.empty(key.shape, dtype=k.dtype, device=dev)
    if tokens == 0:
        return q_out, k_out
    with _lib.on_device(dev):
        _lib.call("bfa_qk_norm_rope", q.data_ptr(), q.shape[1], q.stride(0), q.stride(1), q_out.data_ptr(),
                  k.data_ptr(), k.shape[1], k.stride(0), k.stride(1), k_out.data_ptr(), code, tokens, dim,
                  _lib.ptr(weights[0]), _lib.ptr(weights[1]), w_code, float(eps), positions.data_ptr(),
                  _lib.dtype_code(positions), cos_sin_cache.data_ptr(), max_position,
                  _lib.status_word(dev).data_ptr(), _lib.stream_of(dev))
    return q_out, k_out
