"""Plain 64-bit restatements for the paged serving operators, and their inputs."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from tests.helpers import gen

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def to_fp4(x: torch.Tensor):
    """(codes, scale bytes) of x [..., D], from the definition, block by block in 64 bits."""
    b = x.double().unflatten(-1, (-1, 32))
    most = b.abs().amax(-1)
    e = torch.full_like(most, -126)
    for k in range(-126, 128):  # the smallest power of two that keeps `most` within 6
        e = torch.where(most > 6 * 2.0 ** (k - 1), torch.full_like(e, k), e)
    finite = torch.isfinite(b).all(-1)
    e = torch.where(finite, e, torch.zeros_like(e))
    y = torch.where(finite[..., None], b / torch.exp2(e)[..., None], torch.zeros_like(b))
    gap = (y.abs()[..., None] - LEVELS).abs()
    near = gap.amin(-1, keepdim=True)
    odd = torch.tensor([0, 1] * 4)
    code = torch.where(gap == near, odd, 2).argmin(-1)  # of two equally near the even code
    code = code + 8 * (torch.signbit(y) & (y != 0))
    code = code.flatten(-2)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255))
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def from_fp4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float64 values of codes and scale bytes."""
    c, s = codes.cpu().long(), scales.cpu().double()
    code = torch.stack((c % 16, c // 16), -1).flatten(-2)
    v = LEVELS[code % 8] * (1 - 2 * (code // 8))
    scale = torch.where(s == 255, torch.full_like(s, math.nan), torch.exp2(s - 127))
    return (v.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def make_batch(seed, seq_lens, query_lens, page_size, spare=2):
    """Page lists (host tensors) of the requests over shuffled pages."""
    g = gen(seed)
    pages = [-(-n // page_size) for n in seq_lens]
    total = sum(pages)
    perm = torch.randperm(total + spare, generator=g).to(torch.int32)
    off = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32)  # noqa: E731
    return SimpleNamespace(
        seq=list(seq_lens), query=list(query_lens), num_pages=total + spare, page_size=page_size,
        kv_indices=perm[:total].contiguous(), kv_indptr=off(pages), qo_indptr=off(query_lens),
        last=torch.tensor([n - (p - 1) * page_size if p else 0 for n, p in zip(seq_lens, pages)], dtype=torch.int32),
        tokens=sum(query_lens))


def request_rows(cache, batch, s):
    """K and V [tokens, Hkv, D] of request s; cache: float64 HND [pages, 2, Hkv, slots, D]."""
    ids = batch.kv_indices[int(batch.kv_indptr[s]): int(batch.kv_indptr[s + 1])].long()
    rows = cache[ids].permute(1, 0, 3, 2, 4).flatten(1, 2)[:, : batch.seq[s]]  # [2, tokens, Hkv, D]
    return rows[0], rows[1]


def attention64(q, cache, batch, scale, window=None, sinks=0):
    """(out, allowance parts) in float64 on q's device.  The parts, of out's shape:
    `a` = sum_j p |v| / sum_j p, `s` = the largest scale sum_d |q| |k| of the row's visible
    keys, `v` = sum_j |v| / sum_j exp(score - max) over them."""
    t, hq, d = q.shape
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    a, s_max, v_sum = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    group = hq // cache.shape[2]
    for s in range(len(batch.seq)):
        n, m, at = batch.seq[s], batch.query[s], int(batch.qo_indptr[s])
        if n == 0 or m == 0:
            continue
        k, v = (x.repeat_interleave(group, 1).permute(1, 0, 2) for x in request_rows(cache, batch, s))
        x = q[at: at + m].double().permute(1, 0, 2)
        z = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
        p = torch.arange(n - m, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        seen = j <= p
        if window is not None:
            seen = seen & ((p - j < window) | (j < sinks))
        z = z.masked_fill(~seen, -math.inf)
        top = z.amax(-1, keepdim=True)
        w = torch.exp(z - torch.where(torch.isneginf(top), torch.zeros_like(top), top))
        w = torch.where(seen, w, torch.zeros_like(w))
        total = w.sum(-1, keepdim=True)
        safe = torch.where(total == 0, torch.ones_like(total), total)
        vv = torch.where(seen.any(0)[None, :, None], v, torch.zeros_like(v))
        for h in range(hq):  # a key that a row does not see must not reach it, a NaN among them
            out[at: at + m, h] = _weighted(w[h], vv[h]) / safe[h]
            a[at: at + m, h] = _weighted(w[h], vv[h].abs()) / safe[h]
            v_sum[at: at + m, h] = _weighted(seen.double(), vv[h].abs()) / safe[h]
        s_abs = torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()) * abs(scale)
        s_max[at: at + m] = torch.where(seen, s_abs, torch.zeros_like(s_abs)).amax(-1).permute(1, 0)[..., None]
    return out, (a, s_max, v_sum)


def _weighted(w, v):
    if torch.isfinite(v).all():
        return w @ v
    bad = ~torch.isfinite(v)
    o = w @ torch.where(bad, torch.zeros_like(v), v)
    for j in bad.any(1).nonzero()[:, 0].tolist():
        seen = w[:, j] > 0
        o[seen] += w[seen, j, None] * torch.where(bad[j], v[j], torch.zeros_like(v[j]))
    return o


def attention_allowance(out64, parts, dtype, tiles):
    """How far a kernel may be from `out64`, element by element.  u is half a step of the
    16-bit type.  The weights are rounded to it (u a) and so is the result (u |out|, and u
    of what the first added); a score is a sum of D <= 128 exact products in fp32, off by
    at most 128 x 2^-24 of the products' magnitudes, which moves its weight, and the
    normalisation, by that share (2 s 2^-17 a; in base 2 the scaled score is rounded three
    times more, 3 x 2^-24 of it: within the same term doubled); exp2, the sums over the
    keys of each tile and the rescaling between tiles are off by a few 2^-24 of a for each
    tile.  A weight below fp16's normal range is off by 2^-25 at most."""
    a, s, v = parts
    u = half_step(dtype)
    allow = (u + u * u) * a + u * out64.abs() + (4 * s * 2.0 ** -17 + (tiles + 16) * 2.0 ** -21) * a
    if dtype == torch.float16:
        allow = allow + 2.0 ** -25 * v + 2.0 ** -25
    return allow
